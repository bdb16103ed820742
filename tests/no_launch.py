"""The entry points on the CPU with the launches left out: what they check, save and refuse before and behind one.
Results are whatever the output memory holds."""
import pytest

from hopper_megamoe_basedondeepgemm_amd import _lib

LAUNCHES = ("dgm_rms_norm_residual", "dgm_rms_norm_residual_backward", "dgm_int8_gemm_nt", "dgm_router_balance_loss",
            "dgm_router_balance_loss_backward")


class Library:
    """The built library; LAUNCHES are counted and return 0 (or the status they are given)."""

    def __init__(self, lib):
        self.lib, self.calls, self.status = lib, [], 0

    def __getattr__(self, name):
        if name not in LAUNCHES:
            return getattr(self.lib, name)

        def launch(*args):
            self.calls.append(name)
            return self.status
        return launch


@pytest.fixture
def no_launch(monkeypatch):
    library = Library(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: library)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setattr(_lib, "require_one_device", lambda *tensors: None)
    monkeypatch.setattr(_lib, "no_graph_under_capture", lambda: None)
    return library
