"""A last turn of the 8-bit product's pairs in half tiles: second halves that have columns, behind whole tiles over several blocks of K, for each type of result, on 16 bytes and off them."""
import pytest
import torch

from test_gemm_int8_edges_gpu import whole
from test_gemm_int8_gpu import DT


def halves(m, n, k, pairs):
    """How the product chooses its column tiles, restated: whether they have 256 columns and the last turn's are taken as two each."""
    alone, busy = (112, 138, 194, 265), (208, 277, 347, 417)
    row_tiles, blocks, found = -(-m // 256), -(-k // 128), []
    across = -(-k // 16) * 16 % 128 != 0
    for bn in (256, 192, 128, 64):
        tiles = row_tiles * -(-n // bn)
        turns, left = -(-tiles // pairs), tiles % pairs
        turn = max(blocks * (busy if turns > 1 else alone)[bn // 64 - 1] * (4 if across else 3) // 3, 300 + 9 * bn)
        split = bn == 256 and turns > 1 and left > 0 and 2 * left <= pairs
        found.append((4000 + 6 * bn + turns * turn - (turn // 3 if split else 0), -bn, split))
    return min(found)[2]


# second halves of the last column tile with 116, 104, 66, 83, 128, 2 and 1 columns, several blocks of K, rows of operands on 128 bytes and off them
HALVES = [(6656, 1012, 1024), (10240, 1000, 1000), (6245, 962, 1024), (6163, 979, 793), (6656, 1024, 900), (12879, 386, 777), (12562, 385, 777)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("m,n,k", HALVES)
def test_a_last_turn_in_half_tiles(built_lib, m, n, k, dt):
    assert torch.cuda.get_device_properties(0).multi_processor_count == 148  # 74 pairs of CTAs
    assert halves(m, n, k, 74)
    whole(m, n, k, dt, "wide", [(0, n + 1), (3, n + 4), (16, -(-n // 16) * 16 + 32)])


def test_the_rule_is_that_of_the_source():
    """The numbers that the product chooses its tiles by, as they stand in its source."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_b200", "csrc", "gemm_int8.cu")).read()
    rule = re.sub(r"//[^\n]*", "", text[text.index("Width pair_width("):text.index("int launch_pairs(")])
    for part in ("alone_ns[4] = {112, 138, 194, 265}, busy_ns[4] = {208, 277, 347, 417}", "results = 300 + 9 * bn", "halves = bn == BN && turns > 1 && left > 0 && 2 * left <= pairs",
                 "ns = 4000 + 6 * bn + turns * turn - (halves ? turn / 3 : 0)", "kb * block * (across ? 4 : 3) / 3"):
        assert part in rule, part
