"""The example trains, and decodes what its whole pass computes."""

import pytest

pytestmark = pytest.mark.gpu


def test_block_layer(gpu):
    from nacho_amd.examples import block_layer

    losses, apart = block_layer.main(["--steps", "160"])
    # from about log(64) to what a layer that finds the earlier token leaves
    assert losses[0] > 3.5 and losses[-1] < 0.5
    # float32 throughout: a whole pass and a step sum in another order
    assert apart < 1e-3
