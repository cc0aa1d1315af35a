"""When a session reads shared prefixes apart: the rule alone, no GPU needed."""
import pytest

from richengine_b200.abi import BF16, FP8E4M3, INT4, INT8, Layout
from richengine_b200.session import TILE_PRICE, DecodeSession, prefix_saving

FORMATS = [INT4, INT8, FP8E4M3, BF16]


def layout(fmt):
    return Layout(1, 4, 256, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_pair_saves_nothing_at_any_length(fmt):
    assert prefix_saving(layout(fmt), [(2, 8192)]) < 0
    assert prefix_saving(layout(fmt), [(2, 256)] * 512) < 0
    assert prefix_saving(layout(fmt), []) == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_group_the_search_may_form_saves_something(fmt):
    """Groups start at one lane more than a tile's price; a second and a third tile (22 and 43 lanes) do not turn that round."""
    for lanes in range(int(TILE_PRICE[fmt]) + 1, 1025):
        assert prefix_saving(layout(fmt), [(lanes, 1)]) > 0, lanes


def test_measured_batches_fall_on_the_faster_side():
    """(format, lanes of a group, groups, tokens shared, us with shared prefixes, us without), on a B200. A batch whose two times are
    within 5 % may fall on either side; one that the rule leaves alone may lose what it could have gained, none loses by it."""
    measured = [(INT4, 4, 1, 65536, 59.7, 58.8), (INT4, 6, 1, 4096, 30.8, 23.7), (INT4, 6, 1, 65536, 62.0, 79.5), (INT4, 8, 1, 4096, 31.5, 24.8),
                (INT4, 8, 1, 65536, 64.8, 101.4), (INT4, 4, 32, 8192, 176.0, 148.2), (INT4, 8, 16, 8192, 112.1, 156.3), (INT4, 21, 6, 8192, 72.7, 151.9),
                (INT4, 24, 6, 8192, 91.8, 170.6), (INT4, 32, 1, 8192, 52.0, 61.0), (INT8, 3, 32, 8192, 210.6, 183.6), (INT8, 6, 1, 4096, 29.8, 23.9),
                (INT8, 8, 1, 16384, 39.0, 46.6), (INT8, 8, 16, 8192, 138.2, 230.4), (FP8E4M3, 3, 32, 8192, 233.9, 182.2), (FP8E4M3, 4, 32, 8192, 235.8, 232.4),
                (FP8E4M3, 8, 1, 16384, 41.4, 48.2), (FP8E4M3, 8, 16, 8192, 145.5, 229.6), (BF16, 2, 64, 8192, 547.9, 444.9), (BF16, 3, 1, 16384, 40.9, 35.2),
                (BF16, 3, 32, 8192, 300.8, 337.0), (BF16, 4, 1, 16384, 41.7, 39.4), (BF16, 8, 1, 4096, 33.1, 31.2), (BF16, 8, 1, 16384, 45.8, 64.2),
                (INT4, 5, 24, 8192, 158.2, 139.8), (INT4, 6, 20, 8192, 124.4, 145.7), (INT4, 16, 1, 8192, 38.8, 37.8), (INT4, 16, 1, 16384, 44.2, 59.1),
                (INT8, 32, 1, 2048, 40.4, 31.6), (INT8, 16, 1, 8192, 38.9, 45.7), (FP8E4M3, 32, 1, 2048, 41.6, 35.0), (FP8E4M3, 5, 24, 8192, 211.4, 211.9),
                (BF16, 16, 1, 2048, 33.6, 29.4), (BF16, 32, 1, 2048, 41.8, 40.4), (BF16, 6, 1, 8192, 35.2, 35.3), (BF16, 43, 3, 8192, 131.6, 359.2)]
    for fmt, lanes, groups, tokens, shared, plain in measured:
        formed = lanes > TILE_PRICE[fmt]
        worth = DecodeSession.kWorthBytes + min(lanes * groups, 32) * DecodeSession.kWorthLaneBytes
        used = formed and prefix_saving(layout(fmt), [(lanes, tokens // 32)] * groups) >= worth
        assert not used or shared <= 1.05 * plain, (fmt, lanes, groups, tokens)
        assert used or plain <= 1.15 * shared, (fmt, lanes, groups, tokens)
