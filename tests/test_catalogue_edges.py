"""CPU tests of what the catalogue operators and the factor models refuse, before any library call."""
import numpy as np
import pytest

from recommenders_amd.models import BPR, MF, WMF


@pytest.mark.parametrize("model", [BPR, MF, WMF])
def test_models_without_factors(model):
    for m in (model(), model(init_params={"U": np.zeros((3, 2), np.float32)})):
        for call in (lambda: m.log_prob([0], [[0]]), lambda: m.fit_preferences([0], [[0]], [[1]]), lambda: m.fit_policy([0], [[0]], [1.0])):
            with pytest.raises(RuntimeError, match="has no factors: pass init_params"):
                call()
