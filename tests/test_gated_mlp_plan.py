"""Which kernels the feed-forward block's products are sent to, seen in the
workspace that they ask for (no device work).  The forward pass's holds h and,
where a product runs on the DMA tiles in several parts of k, their fp32 sums."""
import pytest

from pih_amd import abi
from tests.test_adapter_loss_refusals import _query


def _sums(rows, inter, hidden):
    code, need = _query(abi.WORKSPACE_GATED_MLP, rows, inter, hidden)
    assert code == abi.OK
    h = -(-rows * inter * 2 // 256) * 256
    assert need >= h
    return need - h


@pytest.mark.parametrize("rows,inter,hidden", [(65, 5696, 2048), (130, 4160, 1024), (192, 12352, 4096), (130, 8256, 4096),
                                               (17, 12352, 4096), (64, 16448, 64)])
def test_down_stays_split_where_no_tile_takes_its_sizes(rows, inter, hidden):
    """Half a step of 128 behind the last whole one: the tiles chosen per shape do
    not take down, and it would run unsplit on tiles that leave most CUs idle
    (192 rows of 12352 -> 4096 152 us, 104 in parts)."""
    assert inter % 128 == 64
    planes = _sums(rows, inter, hidden) / (rows * hidden * 4)
    assert planes >= 2


@pytest.mark.parametrize("rows,inter,hidden", [(1, 12352, 4096), (8, 12352, 4096), (57, 2112, 4096), (57, 2048, 4096),
                                               (8, 12288, 4096)])
def test_few_rows_take_no_sums(rows, inter, hidden):
    """(the GEMV, or the tiles chosen per shape)"""
    assert _sums(rows, inter, hidden) == 0
