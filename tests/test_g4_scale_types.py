"""G4Weights and the types that scales may have, before anything reaches the device."""
import numpy as np
import pytest

from rknpu2_matmul_open_amd import capi, ops
from tests.test_mx4_wrappers import Session


@pytest.mark.parametrize("scale_type", [capi.MX4_F32, 3, -1, "float16"])
def test_other_scale_types_are_refused_in_words(scale_type):
    s = Session()
    with pytest.raises(TypeError, match="scales of float16 or bfloat16"):
        ops.G4Weights(s, 64, 4, 32, np.zeros((4, 32), np.uint8), np.zeros((4, 2), np.float16), scale_type=scale_type)
    assert not s.lib.calls
