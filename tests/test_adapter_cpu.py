"""Refusals of the adapted projection (kge/adapter.py): every check of an argument comes before the
check of the device, so they are all reached with CPU tensors and no launch."""
import ctypes

import pytest
import torch

from kge import _lib as L
from kge import engine
from kge.adapter import LowRankAdapters


def _args(n=5, d=8, m=6, k=3, r=2, dtype=torch.float32):
    return dict(x=torch.randn(n, d).to(dtype), w=torch.randn(m, d).to(dtype), a=torch.randn(k, r, d).to(dtype),
                b=torch.randn(k, m, r).to(dtype), ids=torch.tensor([0, 2, -1, 1, 0][:n]), scales=torch.ones(k))


def test_cpu_tensors_are_refused_after_the_arguments():
    for dtype in (torch.float32, torch.bfloat16):
        with pytest.raises(L.EngineError, match="MI355X"):
            engine.adapted_projection(**_args(dtype=dtype))
    with pytest.raises(L.EngineError, match="MI355X"):
        LowRankAdapters(3, 2, 8, 6)(torch.zeros(5, 8), torch.zeros(6, 8), torch.zeros(5, dtype=torch.int64))


@pytest.mark.parametrize("change, what", [
    (dict(x=torch.zeros(5, 8, dtype=torch.float16)), "x"), (dict(x=torch.zeros(5, 8, 1)), "x"),
    (dict(w=torch.zeros(6, 8, dtype=torch.bfloat16)), "w"), (dict(w=torch.zeros(6, 9)), "w"),
    (dict(w=torch.zeros(6, 8, requires_grad=True)), "frozen"), (dict(w=torch.zeros(0, 8), b=torch.zeros(3, 0, 2)), "m=0"),
    (dict(a=torch.zeros(2, 8)), "a"), (dict(a=torch.zeros(3, 2, 7)), "a"), (dict(b=torch.zeros(3, 2, 6)), "b"),
    (dict(b=torch.zeros(4, 6, 2)), "b"), (dict(a=torch.zeros(3, 0, 8), b=torch.zeros(3, 6, 0)), "r=0"),
    (dict(a=torch.zeros(1, 1025, 8), b=torch.zeros(1, 6, 1025)), "r=1025"),
    (dict(ids=torch.zeros(4, dtype=torch.int64)), "ids"), (dict(ids=torch.zeros(5)), "ids"),
    (dict(ids=torch.zeros(5, 1, dtype=torch.int64)), "ids"), (dict(scales=torch.ones(2)), "scales"),
    (dict(scales=torch.ones(3, dtype=torch.int64)), "scales"), (dict(scales=torch.ones(3, requires_grad=True)), "scales")])
def test_arguments_refused(change, what):
    with pytest.raises(ValueError, match=what):
        engine.adapted_projection(**{**_args(), **change})


@pytest.mark.parametrize("bad", [-2, 3])
def test_ids_out_of_range_refused_under_index_checking(bad):
    with pytest.raises(IndexError, match="adapter id"):
        engine.adapted_projection(**{**_args(), "ids": torch.tensor([0, 1, bad, -1, 2])})


@pytest.mark.parametrize("args", [(0, 2, 8, 6), (3, 0, 8, 6), (3, 1025, 8, 6), (3, 2, 0, 6), (3, 2, 8, 0)])
def test_module_sizes_refused(args):
    with pytest.raises(ValueError):
        LowRankAdapters(*args)


def test_a_new_adapter_changes_nothing_and_scales_follow_alpha():
    mod = LowRankAdapters(3, 4, 8, 6, alpha=8.0)
    assert (mod.b == 0).all() and (mod.scales == 2.0).all() and mod.a.shape == (3, 4, 8) and mod.b.shape == (3, 6, 4)
    assert set(mod.state_dict()) == {"a", "b", "scales"}


def test_c_entries_refuse_bad_shapes_without_a_device():
    lib = L.lib()
    assert lib.kge_adapter_save_size(4, 8, 3, 0) == 0 and lib.kge_adapter_save_size(-1, 8, 3, 2) == 0
    assert lib.kge_adapter_backward_ws_size(2, 4, 8, 6, 3, 2, 1, 1, 1) == 0
    for want in ((0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1)):  # any choice of gradients has a size
        assert lib.kge_adapter_backward_ws_size(0, 4, 8, 6, 3, 2, *want) >= 0
    size = lib.kge_adapter_save_size(4, 8, 3, 2)
    save = ctypes.create_string_buffer(size + 16)
    at = (ctypes.addressof(save) + 15) // 16 * 16

    def forward(dtype=0, ldx=8, d=8, m=6, k=3, r=2, save=at, size=size):
        return lib.kge_adapter_forward(None, dtype, ldx, 4, d, None, 8, m, None, None, k, r, None, None, None, 6, save, size,
                                       0, None, 0, None)

    # null tensors, types, strides, sizes, workspaces: a status, never an exception
    assert {forward(), forward(dtype=2), forward(ldx=7), forward(m=0), forward(k=0), forward(r=1025),
            forward(save=None), forward(save=at + 4), forward(size=size - 1)} == {1001}
    assert lib.kge_adapter_backward(None, 0, 6, 4, 6, None, 8, 8, None, 8, None, None, 3, 2, None, at, size, None, 8, None,
                                    None, None, 0, None) == 1001


def test_workspace_of_a_backward_pass_does_not_grow_with_the_adapters():
    """Slabs are for adapters of more rows than a chunk, of which there are few however many adapters there are; only
    the transposed adapters of dx take room for each (k r d elements)."""
    size = lambda k, dx: L.lib().kge_adapter_backward_ws_size(0, 5000, 64, 1000, k, 8, dx, 1, 1)  # noqa: E731
    assert size(100000, 0) <= size(10, 0)  # (u's partial sums: fewer with more adapters)
    assert size(100000, 1) <= size(10, 1) + 100000 * 8 * 64 * 4


def test_long_sums_of_few_rows_take_a_workspace():
    """A sum of many products for few results is split over workgroups (slabs in fp32), forwards and for dx."""
    forward = lambda *a: L.lib().kge_adapter_forward_ws_size(*a)  # noqa: E731
    assert forward(0, 100, 40000, 64, 3, 4, 1) >= 2 * 100 * 64 * 4
    assert forward(0, 20, 40000, 64, 3, 4, 0) == 0  # few requests: no tiles
    assert forward(1, 1024, 512, 14541, 64, 16, 1) == 0 and forward(1, 0, 40000, 64, 3, 4, 1) == 0
    back = lambda dx: L.lib().kge_adapter_backward_ws_size(0, 100, 64, 40000, 3, 4, dx, 0, 0)  # noqa: E731
    assert back(1) >= back(0) + 2 * 100 * 64 * 4


def test_few_requests_need_no_workspace():
    from kge.adapter import FEW
    for n in (FEW, FEW + 1):
        assert (L.lib().kge_adapter_forward_ws_size(0, n, 40000, 64, 3, 4, 0) == 0) == (n == FEW)
