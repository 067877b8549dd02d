"""Who asks whether a bounded wait of the linear map's kernels ran out, on the CPU."""
import pytest
import torch

from qkan_b200 import QKAN, _abi
from qkan_b200 import functional as F


class OnTheHost(QKAN):
    """The head alone, by torch: train_ needs nothing else of a model."""

    def forward(self, x):
        for layer in list(self.layers)[1:]:
            x = x if isinstance(layer, torch.nn.Identity) else torch.nn.functional.linear(x, layer.weight, layer.bias)
        return x


def _train(monkeypatch, steps, log, fused=True, fail_at=None):
    asked = []

    def status(device=None):
        asked.append(torch.device(device).type)
        if fail_at is not None and len(asked) == fail_at:
            raise _abi.QkanLibraryError("3 waits ran out")

    monkeypatch.setattr(F, "dense_status", status)
    model = OnTheHost([3, 4, 2], is_map=True, hidden=5, fused_head=fused, device="cpu", seed=0)
    if not fused:
        model.layers[2] = torch.nn.Identity()
    data = {k: torch.randn(8, 3 if k.endswith("input") else 2) for k in ("train_input", "train_label", "test_input", "test_label")}
    data["train_input"], data["test_input"] = torch.randn(8, 4), torch.randn(8, 4)
    try:
        model.train_(data, steps=steps, log=log, verbose=False)
    finally:
        model.asked = asked
    return asked


@pytest.mark.parametrize("steps,log,times", [(6, 1, 6), (6, 3, 3), (7, 3, 3), (1, 5, 1), (4, 0, 4), (0, 1, 0)])
def test_training_asks_at_log_steps_and_at_the_end(monkeypatch, steps, log, times):
    asked = _train(monkeypatch, steps, log)
    assert asked == ["cpu"] * times


def test_training_stops_where_a_wait_ran_out(monkeypatch):
    with pytest.raises(_abi.QkanLibraryError, match="ran out"):
        _train(monkeypatch, 6, 1, fail_at=2)


def test_models_without_dense_modules_do_not_ask(monkeypatch):
    assert _train(monkeypatch, 3, 1, fused=False) == []
