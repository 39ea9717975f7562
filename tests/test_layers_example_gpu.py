"""The example that runs the layer operators together: adapters beside a
protected low-precision model learn from its teacher's top logits, then a
batch of requests decodes."""
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", ["fp8", "nvfp4"])
def test_adapters_recover_part_of_the_quantisation_loss(precision):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import distill_adapters

    args = distill_adapters.parser().parse_args(
        ["--precision", precision, "--steps", "20", "--requests", "4", "--sequence", "64", "--hidden", "256",
         "--vocab", "2048"])
    before, after, detections, gemms, decoded = distill_adapters.train(args)
    assert 0 < after < before
    assert detections == 0 and gemms > 0
    assert decoded.shape == (4, 4) and (decoded >= 0).all() and (decoded < 2048).all()
