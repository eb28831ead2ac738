"""The order in which the weights' tile kernel hands its sums to the two groups of warps that add them
up, worked through on the host: every group follows every phase of the barriers it waits on, and no
barrier can be a phase further than the one that is waited for."""
import pytest

SUMS = 3                             # places for sums in tensor memory


def order(tiles, rtiles, first_row_tile, u0, u1):
    """The group of every sum of a CTA with units u0 .. u1 - 1 (tile u % tiles of a head):
    two tiles at a time where both are one head's, else one whose sums alternate."""
    out, u = [], u0
    while u < u1:
        t = u % tiles
        two = u + 1 < u1 and t + 1 < tiles
        for _ in range(first_row_tile(t), rtiles):
            if two:
                out += [0, 1]
            else:
                out.append(len(out) & 1)
        u += 1 + two
    return out


def by_place(groups):
    """A barrier a place, phase di / SUMS: what a group that skips the other's sums would see."""
    return [(di % SUMS, di // SUMS) for di in range(len(groups))]


def by_group(groups):
    """Two barriers a group in turn, as the kernel has them."""
    n, out = [0, 0], []
    for g in groups:
        out.append(((g, n[g] & 1), n[g] >> 1))
        n[g] += 1
    return out


def follows_every_phase(groups, waits):
    seen = {}
    for g, (bar, phase) in zip(groups, waits):
        if seen.get((g, bar), -1) + 1 != phase:
            return False
        seen[g, bar] = phase
    return True


def never_a_phase_too_far(groups, waits):
    """Sum di is issued once sum di - SUMS has been left; a group leaves its sums in order. With a group
    held before its sum `at`, all that can be issued: is the phase after the one it waits for?"""
    for at, g in enumerate(groups):
        for di in range(at + 1, len(groups)):
            if di - SUMS >= at and any(groups[x] == g for x in range(at, di - SUMS + 1)):
                break
            if waits[di][0] == waits[at][0]:
                return False
    return True


CASES = [(tiles, rtiles, step, u0, n) for tiles in (1, 2, 3, 5, 8) for rtiles in (1, 2, 3, 4)
         for step in (0, 1) for u0 in (0, 1, 2, 3) for n in (1, 2, 3, 5, 9)]


def test_every_group_follows_every_phase():
    for tiles, rtiles, step, u0, n in CASES:
        g = order(tiles, rtiles, lambda t: min(step * t, rtiles - 1), u0, u0 + n)
        assert all(g[i:i + 3] != [g[i]] * 3 for i in range(len(g) - 2)), (tiles, rtiles, step, u0, n)
        w = by_group(g)
        assert follows_every_phase(g, w) and never_a_phase_too_far(g, w), (tiles, rtiles, step, u0, n)


@pytest.mark.parametrize("groups", [[0, 1] * 6, [0, 1, 0, 0, 1, 0, 1]])
def test_a_barrier_a_place_is_not_followed(groups):
    assert not follows_every_phase(groups, by_place(groups))
