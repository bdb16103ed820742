"""``no_launch`` for the MXFP4 operators and layer norm too."""
import pytest

from hopper_megamoe_basedondeepgemm_amd import _lib
from tests import no_launch

LAUNCHES = no_launch.LAUNCHES + ("dgm_layer_norm_residual", "dgm_layer_norm_residual_backward", "dgm_mxfp4_quantize",
                                 "dgm_mxfp4_gemm_nt", "dgm_mxfp4_linear", "dgm_mxfp4_linear_backward")


class Library(no_launch.Library):
    def __getattr__(self, name):
        if name not in LAUNCHES:
            return getattr(self.lib, name)

        def launch(*args):
            self.calls.append(name)
            return self.status
        return launch


@pytest.fixture
def launches(monkeypatch):
    library = Library(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: library)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setattr(_lib, "require_one_device", lambda *tensors: None)
    monkeypatch.setattr(_lib, "no_graph_under_capture", lambda: None)
    return library
