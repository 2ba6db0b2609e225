"""Refusals of the label losses (kge/label_losses.py): every check of an argument comes before the
check of the device, so they are all reached with CPU tensors and no launch."""
import math

import pytest
import torch

from kge import _lib as L
from kge import engine


def _block(n=4, m=9):
    return torch.randn(n, m), torch.tensor([0, 3, -1, 8][:n])


def _policy(s, y, **kw):
    n = y.numel()
    args = {"advantages": torch.ones(n), "old_logp": torch.zeros(n), "ref_logp": torch.zeros(n)}
    call = {k: kw.pop(k, v) for k, v in args.items()}
    return engine.policy_loss(s, y, call["advantages"], call["old_logp"], call["ref_logp"], **kw)


def test_cpu_tensors_are_refused_after_the_arguments():
    s, y = _block()
    ptr = torch.tensor([0, 2, 4])
    for call in (lambda: engine.label_logprobs(s, y), lambda: _policy(s, y),
                 lambda: engine.preference_loss(s, y, ptr),
                 lambda: engine.policy_loss_grad(s, y, torch.ones(4), torch.zeros(4)),
                 lambda: engine.preference_loss_grad(s, y, ptr)):
        with pytest.raises(L.EngineError, match="MI355X"):
            call()


@pytest.mark.parametrize("scores", [torch.zeros(3), torch.zeros(2, 3, 4), torch.zeros(4, 0),
                                    torch.zeros(4, 9, dtype=torch.float64), torch.zeros(4, 9, dtype=torch.int32)])
def test_score_blocks_refused(scores):
    y = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="scores"):
        engine.label_logprobs(scores, y)


@pytest.mark.parametrize("labels", [torch.zeros(3, dtype=torch.int64), torch.zeros(4, 1, dtype=torch.int64),
                                    torch.zeros(4), torch.zeros(4, dtype=torch.bool)])
def test_labels_refused(labels):
    with pytest.raises(ValueError, match="labels"):
        engine.label_logprobs(torch.zeros(4, 9), labels)


@pytest.mark.parametrize("bad", [-2, 9])
def test_labels_out_of_range_refused_under_index_checking(bad):
    y = torch.tensor([0, 3, -1, bad])
    with pytest.raises(IndexError, match="label"):
        engine.label_logprobs(torch.zeros(4, 9), y)


@pytest.mark.parametrize("temperature", [0.0, -1.0, math.inf, math.nan])
def test_temperature_refused(temperature):
    s, y = _block()
    with pytest.raises(ValueError, match="temperature"):
        engine.label_logprobs(s, y, temperature)
    with pytest.raises(ValueError, match="temperature"):
        _policy(s, y, temperature=temperature)


@pytest.mark.parametrize("kw, what", [
    ({"advantages": torch.ones(5)}, "advantages"), ({"advantages": torch.ones(4, dtype=torch.int64)}, "advantages"),
    ({"advantages": torch.ones(4, requires_grad=True)}, "advantages"), ({"old_logp": torch.zeros(4, 1)}, "old_logp"),
    ({"ref_logp": None, "kl": 0.1}, "ref_logp"), ({"clip": -0.1}, "clip"), ({"clip": (0.2, math.nan)}, "clip"),
    ({"kl": -1.0}, "kl"), ({"scale": math.inf}, "scale"), ({"weights": torch.ones(3)}, "weights")])
def test_policy_arguments_refused(kw, what):
    s, y = _block()
    with pytest.raises(ValueError, match=what):
        _policy(s, y, **kw)


@pytest.mark.parametrize("ptr", [torch.tensor([0, 2]), torch.tensor([[0, 2, 4]]), torch.tensor([0.0, 2.0, 4.0]),
                                 torch.zeros(0, dtype=torch.int64)])
def test_seq_ptr_refused(ptr):
    s, y = _block()
    with pytest.raises(ValueError, match="seq_ptr"):
        engine.preference_loss(s, y, ptr)


@pytest.mark.parametrize("ptr", [[0, 2, 5], [-1, 2, 4], [0, 3, 2]])
def test_seq_ptr_out_of_range_refused_under_index_checking(ptr):
    s, y = _block()
    with pytest.raises(IndexError, match="seq_ptr"):
        engine.preference_loss(s, y, torch.tensor(ptr))


@pytest.mark.parametrize("kw, what", [({"beta": -1.0}, "beta"), ({"smoothing": 1.5}, "smoothing"),
                                      ({"ref_logp": torch.zeros(3)}, "ref_logp")])
def test_preference_arguments_refused(kw, what):
    s, y = _block()
    with pytest.raises(ValueError, match=what):
        engine.preference_loss(s, y, torch.tensor([0, 2, 4]), **kw)


def test_c_entries_refuse_bad_shapes_without_a_device():
    lib = L.lib()
    assert lib.kge_label_ws_size(-1, 5, 0, 0) == 0 and lib.kge_label_ws_size(5, 0, 0, 0) == 0
    assert lib.kge_label_ws_size(5, 5, 3, 0) == 0 and lib.kge_label_ws_size(5, 5, 0, -1) == 0
    assert lib.kge_label_logprobs(None, 0, 5, 4, 5, None, 1.0, None, None, None, 0, None) == 1001
    assert lib.kge_label_logprobs(None, 7, 5, 0, 5, None, 1.0, None, None, None, 0, None) == 1001
    assert lib.kge_label_logprobs(None, 0, 5, 0, 5, None, 0.0, None, None, None, 0, None) == 1001
    assert lib.kge_label_logprobs(None, 0, 5, 0, 5, None, 1.0, None, None, None, 0, None) == 0  # no rows: nothing to do
    assert lib.kge_label_grad(None, 0, 5, 4, 5, None, 1.0, None, None, None, None, 5, None) == 1001


@pytest.mark.parametrize("n, m, pairs", [(1, 7, 0), (3, 100000, 500), (2047, 14541, 2048), (2049, 14541, 1)])
def test_workspace_covers_parts_rows_and_losses(n, m, pairs):
    """8 + 4 bytes per row, 8 per loss, and where rows are cut into parts (over 64 KiB) 8 for each of them: k
    rows are cut into at most ceil(2048 / k) parts each, for any k <= n."""
    for code, es in ((0, 4), (1, 2), (2, 2)):
        parts = max(k * -(-2048 // k) for k in range(1, n + 1)) if m * es > 65536 else 0
        size = L.lib().kge_label_ws_size(n, m, code, pairs)
        least = n * 8 + n * 4 + max(n, pairs) * 8
        assert least + parts * 8 <= size <= least + (n + 2048) * 8 + 4 * 256


@pytest.mark.parametrize("temperature", [1e-31, 1e31])
def test_temperatures_whose_factor_is_no_32_bit_number_are_refused(temperature):
    """log2(e) / temperature would be infinite (0 * inf is NaN for a row's largest score) or 0 (-inf * 0)."""
    s, y = _block()
    with pytest.raises(ValueError, match="temperature"):
        engine.label_logprobs(s, y, temperature)
    assert L.lib().kge_label_logprobs(None, 0, 5, 0, 5, None, temperature, None, None, None, 0, None) == 1001


def test_seq_ptr_of_booleans_refused():
    s, y = _block()
    with pytest.raises(ValueError, match="seq_ptr"):
        engine.preference_loss(s, y, torch.tensor([False, True, True]))
