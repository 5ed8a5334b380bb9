"""The example layer trains, and answers alike in 8 bits."""

import runpy
from pathlib import Path

import pytest

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "expert_layer.py"


@pytest.mark.gpu
def test_expert_layer_example(gpu):
    main = runpy.run_path(str(EXAMPLE))["main"]
    losses, error = main(steps=40, verbose=False)
    assert losses[-1] < 0.7 * losses[0]
    # both products of 8-bit rows and weights: each rounds values of up to 127
    # steps by half a step, so a result is off by under 3% of its size
    assert error < 0.03
