"""gated_ffn at widths where a product's tiles do not come out even."""
import pytest
import torch

from tests.test_gated_ffn_gpu import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("r,e,f", [(64, 512, 32832), (130, 512, 68864)])
def test_one_row_of_tiles_with_more_columns_than_a_round_of_workgroups(r, e, f):
    """Rows that cannot be parted between two launches stay in one."""
    torch.manual_seed(0)
    _check(_inputs(r, e, f, True), "silu")
