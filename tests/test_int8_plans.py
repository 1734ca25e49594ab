"""How calls on 8-bit integers are cut up, on the host: what the kernels are given bounds what they find."""
import random

import pytest

from gpt_fast_b200.ops.cuda import int8_pairs, int8_plan, int8_shares

SMS = 148


@pytest.mark.parametrize("seed", range(20))
def test_pairs_of_tiles_are_bounded(seed):
    rng = random.Random(seed)
    for _ in range(200):
        rep = rng.choice([1, 2, 3, 4, 5, 8, 16, 40, 128])
        new = [rng.choice([1, 2, 17, 63, 64, 65, 300, 5000]) for _ in range(rng.randint(1, 40))]
        ctx = rng.choice([0, 100, 4000, 100000])
        pairs, even = int8_pairs(sum(new), len(new), max(new), ctx + max(new), rep, rng.choice([1, 2, 8, 40]), SMS)
        two = 2 * (128 // rep)
        assert sum(-(-n // two) for n in new) <= pairs <= sum(-(-n // two) for n in new) + len(new)
        assert not even or pairs <= 1024                      # what a block sorts


def test_shares_where_a_context_is_long_and_items_are_few():
    assert int8_pairs(512, 1, 512, 32513, 4, 8, SMS) == (8, True)
    assert int8_pairs(520, 9, 512, 32513, 4, 8, SMS)[1]       # the same beside decoding sequences
    assert not int8_pairs(2048, 1, 2048, 2048, 4, 8, SMS)[1]
    assert not int8_pairs(60000, 1, 60000, 110000, 4, 8, SMS)[1]


@pytest.mark.parametrize("M", [0, 1, 16, 17, 64, 65, 128, 129, 333, 512, 513, 8192])
def test_products(M):
    for N in (1, 100, 255, 256, 515, 4096, 28672, 131072):
        for K in (1, 100, 4096, 14336, 133144):
            for mode in ("store", "add", "swiglu"):
                bn, splits, stages = int8_plan(M, N, K, mode, SMS)
                assert bn in (16, 32, 64, 128, 256) and 1 <= splits <= 8 and 2 <= stages <= 12
                assert splits == 1 or splits <= -(-K // 128)
                assert bn == 256 or stages * (128 * 128 + bn * 128) <= 227 * 1024 - 2048
                if M and splits > 1:                          # one wave of blocks (no tokens: no blocks)
                    assert -(-N // 128) * -(-M // bn) * splits <= 7 * SMS / 4


def test_single_tokens():
    for longest in (1, 64, 65, 4000, 131072):
        for pairs in (1, 8, 64, 512, 4096, 200000):
            slices, blocks = int8_shares(longest, 64, pairs, SMS)
            assert 1 <= slices <= 8 and blocks in (0, 4 * SMS) and slices <= max(1, -(-longest // 64))
