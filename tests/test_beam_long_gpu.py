"""DeviceBeamSearch.Select on the GPU where a CTA reads many tiles of a row, up to the most that it may."""
import numpy as np
import pytest

from tests.test_beam_gpu import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,k,v,dtype,banned", [
    (38, 8, 131069, "f32", 0.0),   # one CTA a row, 32 tiles of it; rows enough to fill the SMs
    (38, 8, 90001, "bf16", 0.3),   # 11 tiles
    (38, 12, 60001, "f32", 0.0),   # too many beams for a cluster: 15 tiles a part, joined by a second kernel
    (30, 16, 81921, "f16", 0.3)])
def test_many_tiles_a_part(cuda, b, k, v, dtype, banned):
    logits, scores = inputs(b, k, v, dtype, seed=v, banned=banned)
    finished = (np.random.RandomState(v).rand(b, k) < 0.1).astype(np.uint8)
    finished[:, 0] = 0
    check(logits, scores, finished, 5)
