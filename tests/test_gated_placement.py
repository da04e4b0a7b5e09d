"""Every strip of channels of a gated recurrence's call is taken by exactly as many workgroups as it has tiles, for all
ways of placing them on the chip's dies (no GPU needed: the kernels' own mapping, built by a host compiler)."""

from __future__ import annotations

import random

import pytest

from gated_placement import CASES, Shape, build


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    return build(tmp_path_factory.mktemp("tiles"))


def check(tiles, batch, seqlen, dim, backward, ragged):
    s = Shape(tiles, batch, seqlen, dim, backward, ragged)
    blocks = -(-seqlen // 16)
    assert s.strips == batch * -(-dim // 64) and s.waves * s.turns >= blocks > s.waves * (s.turns - 1)
    assert s.waves >= 4 or s.turns == 1  # the waves of a tile that waits share 16 tiles to look back at, 4 each
    assert s.strips % s.span == 0
    count, bad = s.counts(tiles)
    assert bad == 0 and min(count) == max(count) == s.turns, (batch, seqlen, dim, backward, ragged)
    assert s.workgroups <= s.strips * s.turns * 9 / 8
    return s


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_every_tile_is_taken_once(tiles, backward, ragged):
    seen = set()
    for batch in (1, 2, 3, 4, 7, 8, 9, 16, 33, 64):
        for strips in (*range(1, 42), 63, 64, 65, 80, 127, 128):
            for seqlen in (1, 16, 64, 65, 256, 257, 1000):
                s = check(tiles, batch, seqlen, 64 * strips - (strips % 3), backward, ragged)
                seen.add((s.per_die > 0, s.span == s.strips, batch > 1))
    # no placement; by sequence and over all of them (one sequence is both)
    want = {(False, True, False), (False, True, True), (True, True, False), (True, False, True)}
    assert seen == want | (set() if ragged else {(True, True, True)})


def test_random_sizes(tiles):
    rng = random.Random(1)
    for _ in range(300):
        check(tiles, rng.randint(1, 300), rng.randint(0, 3000) or 1, rng.randint(1, 6000), rng.random() < 0.5,
              rng.random() < 0.5)


@pytest.mark.parametrize("size", [(60000, 17, 64 * 2000), (1, 1 << 30, 64 * 60), (9, 1 << 27, 64 * 28)])
def test_many_workgroups(tiles, size):
    """Workgroup numbers next to 2^31: the strips of the last ones, in whole numbers of any size."""
    s = Shape(tiles, *size, True, False)
    assert 10 ** 8 < s.workgroups < 2 ** 31
    for k in range(s.workgroups - 1000, s.workgroups):
        want = k % s.strips
        if s.per_die:
            j, place = k // 8, k % 8 * s.per_die + k // 8 % s.per_die
            want = j // s.per_die * s.span % s.strips + place if place < s.span else -1
        assert tiles.tiles_strip(s.raw, k) == want


@pytest.mark.parametrize("size,per_die", CASES)
def test_cases_of_the_gpu_tests(tiles, size, per_die):
    """The GPU's placement tests run on several sequences whose strips are placed by sequence."""
    for backward in (False, True):
        for ragged in (False, True):
            s = check(tiles, *size, backward, ragged)
            assert s.turns > 1 and s.per_die == per_die and s.span < s.strips
    assert Shape(tiles, *size, False, False).waves == (4 if size[0] == 9 else 8)
