"""The sizes that the adapters' workspaces and grids are made for against what a batch can need: tiles of 64 slots, items
of tiles, partial sums, and 16s of a few rows, counted from the rows of each adapter (without a GPU)."""
import random

import pytest

import nemotron_hip as NH
from dispatch import Recorder
from test_adapters import back_args, lora_args

RANK, N, K = 16, 64, 512


@pytest.fixture
def rec():
    r = Recorder()
    yield r
    r.close()


def up(a, b):
    return -(-a // b)


def item_tiles(m):
    return max(1, (m // 64 + 31) // 32)


def batches(rng, m, adapters):
    """Rows per adapter, the last of them rows without one."""
    it = item_tiles(m)
    for each in (1, 2, 63, 64, 65, 64 * it, 64 * it + 1, 64 * it + 65, 128 * it + 1):
        left, rows = m, []
        for _ in range(adapters):  # as many adapters as there are rows for, the rest to the first or to none
            rows.append(min(each, left))
            left -= rows[-1]
        yield rows + [left]
        yield [rows[0] + left] + rows[1:] + [0]
    yield [m] + [0] * adapters
    yield [0] * adapters + [m]
    for _ in range(4):
        cuts = sorted(rng.randint(0, m) for _ in range(adapters))
        yield [b - a for a, b in zip([0] + cuts, cuts + [m])]


def sizes():
    rng = random.Random(1)
    for adapters in (1, 2, 3, 7, 31, 64, 300, 1023, 1024):
        for m in (1, 2, 15, 16, 17, 33, 63, 64, 65, 127, 129, 1000, 2047, 2048, 2049, 2112, 4095, 4097, 6145, 8192, 8256, 20011,
                  65537, 500000, (1 << 24) - 1, rng.randint(1, 1 << 20)):
            yield rng, m, adapters


def test_what_a_batch_needs_is_there(rec):
    tight = set()
    for rng, m, adapters in sizes():
        small = NH.lib().nh_linear_lora_backward_workspace_size(m, N, K, RANK, adapters)
        large = NH.lib().nh_linear_lora_backward_workspace_size(m, N, 2 * K, RANK, adapters)
        # to 1024 columns shrink has one part, so a wider k makes da's partial sums longer and nothing else
        assert (large - small) % (RANK * K * 4) == 0
        partials = (large - small) // (RANK * K * 4)
        grids = {k: (gx, gy) for k, gx, gy in rec.launches("nh_linear_lora_backward", *back_args(m, N, K, RANK, adapters, h=None))}
        tiles = grids["lora_finish"][0]
        items = grids["lora_outer_bf16_1"][1] // 2
        it = item_tiles(m)
        assert ("lora_reduce" in grids) == (m > 64 * it)
        for rows in batches(rng, m, adapters):
            assert sum(rows) == m
            t = [up(r, 64) for r in rows]
            assert sum(t) <= tiles, (m, adapters, rows)
            i = [up(v, it) for v in t[:-1]]
            assert sum(i) <= items and adapters <= items, (m, adapters, rows)
            p = sum(v for v in i if v > 1)
            assert p <= partials and (p == 0 or m > 64 * it), (m, adapters, rows)
            if m <= 64:
                units = {k: gx for k, gx, _ in rec.launches("nh_linear_lora", *lora_args(m, N, K, RANK, adapters))}
                assert sum(up(r, 16) for r in rows) <= units["lora_shrink_bf16_few_1"] == units["lora_expand_bf16_few_1"]
                tight.add(sum(up(r, 16) for r in rows) == units["lora_shrink_bf16_few_1"])
            # a workgroup of shrink per 16 slots of every tile
            assert 4 * sum(t) <= grids["lora_shrink_bf16_back_1"][0]
    assert True in tight
