"""How attention's backward pass is laid out, on the CPU: columns that are computed."""
import pytest

from train_host import host


@pytest.mark.parametrize("D", range(8, 129, 8))
def test_fp32_computes_the_columns_that_there_are(D):
    """One rule for all head_dims: no column more above 32, none of them a case of its own."""
    assert host().host_f32_groups(D) * 8 == max(D, 32)
