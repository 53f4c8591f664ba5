"""A tree's arrays are freed with its last reference, not when the garbage
collector next runs: an update tree of a large model is most of a GPU."""

import gc
import weakref

import pytest
import torch

from rollfast_b200.tree import MaskedNode, is_aux_leaf, tree_flatten, tree_map, tree_structure_equal, tree_unflatten


def _tree():
    return {"a": torch.zeros(3), "b": [torch.ones(2), (torch.zeros(1), None)], "c": MaskedNode()}


def _drops_flatten(t):
    tree_flatten(t, is_leaf=is_aux_leaf)


def _drops_unflatten(t):
    leaves, treedef = tree_flatten(t)
    tree_unflatten(treedef, list(leaves))


def _drops_map(t):
    tree_map(lambda x, y: x + y, t, t)


def _drops_structure(t):
    tree_structure_equal(t, t)


@pytest.fixture
def no_collector():
    gc.collect()
    gc.disable()
    yield
    gc.enable()


@pytest.mark.parametrize("use", [_drops_flatten, _drops_unflatten, _drops_map, _drops_structure])
def test_arrays_are_freed_with_the_tree(no_collector, use):
    t = _tree()
    refs = [weakref.ref(x) for x in (t["a"], t["b"][0], t["b"][1][0])]
    use(t)
    del t
    assert all(r() is None for r in refs)


@pytest.mark.gpu
@pytest.mark.parametrize("applied", [False, True])
def test_dropped_updates_leave_no_memory_behind(no_collector, applied):
    import rollfast_b200 as rf

    params = {"w": torch.zeros(256, 512, device="cuda"), "v": torch.zeros(4096, device="cuda")}
    grads = {"w": torch.randn(256, 512, device="cuda"), "v": torch.randn(4096, device="cuda")}
    tx = rf.muon(learning_rate=0.02)
    state = tx.init(params)

    def step(state):
        if applied:
            return rf.update_and_apply(tx, grads, state, params, stochastic=False)
        return tx.update(grads, state, params)

    out, state = step(state)
    del out
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        out, state = step(state)
        del out
        assert torch.cuda.memory_allocated() == held


@pytest.mark.gpu
def test_dropped_outputs_of_the_training_step_leave_no_memory_behind(no_collector):
    import rollfast_b200 as rf

    x, g = (torch.randn(300, 264, device="cuda") for _ in range(2))
    w = torch.ones(264, device="cuda")

    def step():
        s = rf.save_activation(x)
        o = rf.block_norm_forward(x, g, pre_weight=w, gate=w, save="int8")
        h, sg, su = rf.swiglu_forward(x, g)
        return (s, rf.load_activation(s), rf.weight_gradient(s, g), o, h, rf.swiglu_backward(h, sg, su, save_h="int8"),
                rf.block_norm_backward(x, g, o.saved_x, o.saved_branch, pre_weight=w, gate=w))

    step()
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        step()
        assert torch.cuda.memory_allocated() == held
