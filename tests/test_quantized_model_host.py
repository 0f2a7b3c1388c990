"""When a linear's packed weight holds, and what quantising a module leaves as it
was, on the CPU."""
import copy
import pickle

import pytest
import torch
import torch.nn as nn
from torch.multiprocessing.reductions import StorageWeakRef

from taomate_amd import dit as D
from taomate_amd import quant

BF = torch.bfloat16
CFG = D.AVConfig(num_layers=1, video_dim=128, audio_dim=64, video_heads=2, audio_heads=1, video_d_head=64,
                 audio_d_head=64)


def _lin():
    return nn.Linear(64, 32, dtype=BF)


def _replace(lin):
    lin.weight = nn.Parameter(lin.weight.detach().clone())


def _in_place(lin):
    with torch.no_grad():
        lin.weight.mul_(2)


def _load(lin):
    lin.load_state_dict({k: v.clone() for k, v in lin.state_dict().items()})


def _assign(lin):
    lin.load_state_dict({k: v.clone() for k, v in lin.state_dict().items()}, assign=True)


def _data(lin):
    lin.weight.data = lin.weight.data.clone()


def _weight_norm(lin):
    nn.utils.parametrizations.weight_norm(lin)


def _dtype(lin):
    lin.float()


@pytest.mark.parametrize("change", [_replace, _in_place, _load, _assign, _data, _weight_norm, _dtype])
def test_a_changed_weight_ends_the_packing(change):
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_mx(lin.weight))
    assert packed.holds(lin)
    change(lin)
    assert not packed.holds(lin)


def test_freed_memory_does_not_come_back_as_the_packed_weight():
    """Weights replaced twice: the first one's memory is held, so no later weight lies there."""
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_mx(lin.weight))
    at = lin.weight.data_ptr()
    for _ in range(50):
        lin.weight.data = torch.randn(32, 64).to(BF)
        assert lin.weight.data_ptr() != at and not packed.holds(lin)


def test_a_new_parameter_over_the_same_memory_ends_the_packing():
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_mx(lin.weight))
    old = lin.weight._version
    lin.weight = nn.Parameter(lin.weight.data)
    for _ in range(old + 2):
        assert not packed.holds(lin)
        with torch.no_grad():
            lin.weight.mul_(2)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda m: pickle.loads(pickle.dumps(m))], ids=["deepcopy", "pickle"])
def test_a_copy_is_not_packed(how):
    """A copy's version count begins anew: changed up to the packed version it must not hold."""
    ff = D.FeedForward(64, 64).to(BF)
    lin = ff.net[2]
    with torch.no_grad():
        lin.weight.mul_(2)
    ff.quantize_()
    two = how(ff)
    assert ff._mx[1].holds(lin)
    for _ in range(lin.weight._version + 2):
        assert not any(p.holds(m) for p, m in zip(two._mx, (two.net[0].proj, two.net[2])))
        with torch.no_grad():
            two.net[0].proj.weight.mul_(2)
            two.net[2].weight.mul_(2)
    with torch.no_grad():
        assert not two.quantized() and two.quantize_() is two


def test_packing_again_keeps_the_memory():
    """What a captured graph reads stays in place and gets the new values; another layout or
    device has memory of its own.  Packing in inference mode makes ordinary tensors."""
    ff = D.FeedForward(64, 64).to(BF)
    with torch.inference_mode():
        ff.quantize_()
    at = [t.data_ptr() for p in ff._mx for t in p.rows.tensors()]
    old = ff._mx[1].rows.dequantize()
    with torch.no_grad():
        ff.net[2].weight.mul_(-3)
    assert not ff._mx[1].holds(ff.net[2]) and ff._mx[0].holds(ff.net[0].proj)
    ff.quantize_()
    assert [t.data_ptr() for p in ff._mx for t in p.rows.tensors()] == at
    assert ff._mx[1].holds(ff.net[2])
    want = quant.quantize_mx(ff.net[2].weight)
    assert torch.equal(ff._mx[1].rows.dequantize(), want.dequantize()) and not torch.equal(want.dequantize(), old)
    lin = nn.Linear(128, 32, dtype=BF)
    D._pack_group4(lin, 32)
    first = lin._group4.rows
    with torch.no_grad():
        lin.weight.neg_()
    D._pack_group4(lin, 32)
    assert lin._group4.rows is first and torch.equal(first.dequantize(), quant.quantize_group4(lin.weight, 32).dequantize())
    D._pack_group4(lin, 64)
    assert lin._group4.rows is not first and lin._group4.rows.group == 64


def test_inference_mode_weights():
    with torch.inference_mode():
        made = _lin()
    with pytest.raises(ValueError, match="inference mode"):
        quant.Packed(made, quant.quantize_mx(made.weight))
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_mx(lin.weight))
    with torch.inference_mode():
        assert packed.holds(lin)
    lin.weight = made.weight
    assert not packed.holds(lin)


def test_quantising_keeps_names_values_and_modules():
    m = D.build_model(CFG, "cpu", seed=1)
    before = {k: v.clone() for k, v in m.state_dict().items()}
    assert m.quantize_linears_(timestep=True, group=64) is m
    after = m.state_dict()
    assert list(after) == list(before) and all(torch.equal(after[k], before[k]) for k in before)
    ff = m.transformer_blocks[0].ff
    assert ff._mx[0].rows.shape == (512, 128) and m.adaln_single.linear._group4.rows.group == 64
    assert m.adaln_single.emb.timestep_embedder.linear_1._group4.rows.shape == (128, 256)
    x = torch.randn(2, 3, 128).to(BF)
    with torch.no_grad():
        assert not ff.quantized() and torch.equal(ff(x), ff.net(x))   # no GPU here: the modules run
    c = copy.deepcopy(m)
    assert torch.equal(c.state_dict()["adaln_single.linear.weight"], before["adaln_single.linear.weight"])
    m.quantize_linears_(feed_forward=False, timestep=False)
    assert "_mx" not in ff.__dict__ and "_group4" not in m.adaln_single.linear.__dict__


def test_what_cannot_be_quantised_is_refused():
    with pytest.raises(ValueError, match="multiple of 32"):
        D.FeedForward(48, 48).to(BF).quantize_()
    with pytest.raises(TypeError, match="plain bf16"):
        D.FeedForward(64, 64).quantize_()
    ff = D.FeedForward(64, 64).to(BF)
    ff.net[2].register_forward_hook(lambda *_: None)
    with pytest.raises(TypeError, match="plain bf16"):
        ff.quantize_()
    with pytest.raises(ValueError, match="at most 8192"):
        D.FeedForward(8224, 32, mult=0.0078125).to(BF).quantize_()
    with pytest.raises(ValueError, match="at most 4096"):
        D._pack_group4(nn.Linear(4224, 8, dtype=BF), 32)
    with pytest.raises(ValueError, match="multiple of 128"):
        D._pack_group4(nn.Linear(64, 8, dtype=BF), 128)


def _packed_at(m):
    return {n: [t.data_ptr() for t in lin._group4.rows.tensors()] for n, lin in m.named_modules() if "_group4" in lin.__dict__}


def test_quantising_again_frees_no_rows():
    """A captured graph reads the packed rows: the documented call after new weights packs all of
    them into the same memory, the 4-bit ones too, in the group that they have."""
    m = D.build_model(CFG, "cpu", seed=1).quantize_linears_(timestep=True, group=64)
    at, lin = _packed_at(m), m.adaln_single.linear
    rows = [r for x in m.modules() if isinstance(x, D.FeedForward) for p in x._mx for r in p.rows.tensors()]
    assert len(at) == 18
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(2)
    assert not lin._group4.holds(lin)
    m.quantize_linears_()
    assert _packed_at(m) == at and lin._group4.holds(lin) and lin._group4.rows.group == 64
    assert torch.equal(lin._group4.rows.dequantize(), quant.quantize_group4(lin.weight, 64).dequantize())
    again = [r for x in m.modules() if isinstance(x, D.FeedForward) for p in x._mx for r in p.rows.tensors()]
    assert all(a is b for a, b in zip(rows, again))
    # a model without 4-bit linears gets none, a copy's are gone with its own first packing
    assert not _packed_at(D.build_model(CFG, "cpu", seed=1).quantize_linears_())
    c = copy.deepcopy(m).quantize_linears_()
    assert not _packed_at(c) and c.transformer_blocks[0].ff._mx[0].holds(c.transformer_blocks[0].ff.net[0].proj)
    # only False ends them
    m.quantize_linears_(timestep=False)
    assert not _packed_at(m) and "_mx" in m.transformer_blocks[0].ff.__dict__
    m.quantize_linears_(timestep=True)
    assert lin._group4.rows.group == 32
    m.quantize_linears_(False)
    assert not _packed_at(m) and "_mx" not in m.transformer_blocks[0].ff.__dict__


class _Elsewhere:
    """Rows as on a GPU, which a graph there may read."""
    def __init__(self, rows):
        self.rows = rows

    def __getattr__(self, name):
        return getattr(self.rows, name)

    @property
    def device(self):
        return torch.device("cuda:0")


def test_another_layout_does_not_replace_rows_on_a_gpu():
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_group4(lin.weight, 32))
    held = packed.rows = _Elsewhere(packed.rows)
    with pytest.raises(ValueError, match="another layout"):
        quant.Packed(lin, quant.quantize_group4(lin.weight, 64), packed)
    assert packed.rows is held
    same = quant.Packed(lin, quant.quantize_group4(lin.weight, 32), packed)
    assert same.rows is held


def test_a_weight_whose_memory_was_exchanged_ends_the_packing():
    """Its storage freed and allocated again elsewhere, as sharded parameters are."""
    lin = _lin()
    packed = quant.Packed(lin, quant.quantize_mx(lin.weight))
    store, at = lin.weight.untyped_storage(), lin.weight.data_ptr()
    size = store.nbytes()
    store.resize_(0)
    assert not packed.holds(lin)
    others = [torch.empty(size, dtype=torch.uint8) for _ in range(8)]   # the old place is taken
    store.resize_(size)
    if any(t.data_ptr() == at for t in others):
        assert lin.weight.data_ptr() != at and not packed.holds(lin)


def _memory(t):
    """A weak reference to a tensor's memory; ``expired()`` once it is freed."""
    return StorageWeakRef(t.untyped_storage())


@pytest.mark.parametrize("change", [_replace, _assign, _data], ids=["parameter", "state dict", "data"])
def test_replaced_weights_are_let_go(change):
    """The first call after a change sees that the packing lapsed and lets go of the old weights;
    the rows, which a captured graph may read, stay until they are dropped."""
    ff = D.FeedForward(64, 64).to(BF).quantize_()
    lins = (ff.net[0].proj, ff.net[2])
    old, rows = [_memory(m.weight) for m in lins], [_memory(t) for p in ff._mx for t in p.rows.tensors()]
    for m in lins:
        change(m)
    with torch.no_grad():
        ff(torch.zeros(2, 64, dtype=BF))
        assert not ff.quantized() and all(m.expired() for m in old) and not any(r.expired() for r in rows)
        assert not any(p.holds(m) for p, m in zip(ff._mx, lins))
        ff.quantize_()
        assert all(p.holds(m) for p, m in zip(ff._mx, lins)) and not any(r.expired() for r in rows)
    ff.quantize_(False)
    assert all(r.expired() for r in rows)


def test_one_replaced_weight_lets_go_of_both():
    ff = D.FeedForward(64, 64).to(BF).quantize_()
    old = _memory(ff.net[0].proj.weight)
    _replace(ff.net[0].proj)
    with torch.no_grad():
        ff(torch.zeros(2, 64, dtype=BF))
    assert old.expired() and not ff._mx[1].holds(ff.net[2])


@pytest.mark.parametrize("part", ["model", "block", "feed-forward", "adaln"])
def test_moved_weights_are_let_go_at_once(part):
    """A model that is cast or moved keeps none of its old weights, whether or not it is called again."""
    m = D.build_model(CFG, "cpu", seed=1).quantize_linears_(timestep=True)
    block = m.transformer_blocks[0]
    of = {"model": m, "block": block, "feed-forward": block.ff, "adaln": m.adaln_single}[part]
    old = [_memory(p) for p in of.parameters()]
    of.to(torch.float32)
    assert len(old) >= 4 and all(r.expired() for r in old)
    of.to(BF)
    with torch.no_grad():
        assert not block.ff.quantized() or part == "adaln"
    m.quantize_linears_()
    assert m.adaln_single.linear._group4.holds(m.adaln_single.linear) and block.ff._mx[0].holds(block.ff.net[0].proj)


def test_replaced_timestep_weights_are_let_go():
    m = D.build_model(CFG, "cpu", seed=1).quantize_linears_(timestep=True)
    lins = [m.adaln_single.linear, m.adaln_single.emb.timestep_embedder.linear_1]
    old = [_memory(x.weight) for x in lins]
    for x in lins:
        _replace(x)
    with torch.no_grad():
        m.adaln_single(torch.zeros(17), BF)
    assert all(r.expired() for r in old)


def test_a_trace_does_not_end_the_packing():
    """Calls that see stand-ins for the weights run the modules and leave the packing as it is."""
    m = D.build_model(CFG, "cpu", seed=1).quantize_linears_(timestep=True)
    emb, ff = m.adaln_single.emb.timestep_embedder, m.transformer_blocks[0].ff
    x, y = torch.zeros(2, 256, dtype=BF), torch.zeros(2, 128, dtype=BF)
    for mod, arg in ((emb, x), (ff, y)):
        other = {k: v.detach().clone() for k, v in mod.named_parameters()}
        torch.func.functional_call(mod, other, (arg,))      # gradients are on
        torch.export.export(mod, (arg,), strict=False)
        with torch.no_grad():
            mod(arg)
    assert emb.linear_1._group4.holds(emb.linear_1) and emb.linear_2._group4.holds(emb.linear_2)
    assert ff._mx[0].holds(ff.net[0].proj) and ff._mx[1].holds(ff.net[2])
