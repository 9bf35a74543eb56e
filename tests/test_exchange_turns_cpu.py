"""The swap of two warps' largest values, tile after tile, in every order in which their steps can come.

A warp writes its values, arrives on its barrier, waits for the phase of the other's barrier and reads the other's values.  A barrier goes
through one phase an arrival, and a wait by parity ends while the number of completed phases is odd (parity 0) or even (parity 1)."""

import pytest

from nanoep_b200.utils.build import load_extension


def _orders(turn_of, tiles):
    """Ends of all orders: what went wrong in them, if anything."""
    wrong, seen, todo = set(), set(), [((0, 0), ((), ()), ((), ()))]
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        at, arrivals, values = state
        stuck = True
        for me, other in ((0, 1), (1, 0)):
            tile, step = divmod(at[me], 4)
            if tile == tiles:
                continue
            place, parity = turn_of(tile)
            now, counts, held = list(at), [dict(a) for a in arrivals], [dict(v) for v in values]
            if step == 0:
                held[me][place] = tile
            elif step == 1:
                counts[me][place] = counts[me].get(place, 0) + 1
            elif step == 2:
                phases = counts[other].get(place, 0)
                if phases % 2 == parity:  # the phase of this parity is not complete, or a later one has taken its place
                    continue
            elif held[other].get(place) != tile:
                wrong.add("values of another tile")
            now[me] += 1
            stuck = False
            todo.append((tuple(now), *(tuple(tuple(sorted(d.items())) for d in both) for both in (counts, held))))
        if stuck and at != (4 * tiles, 4 * tiles):
            wrong.add("a wait that does not end")
    return wrong


@pytest.mark.parametrize("tiles", [1, 2, 3, 7])
def test_every_order_of_the_exchange(tiles):
    assert _orders(load_extension().exchange_turn, tiles) == set()


def test_one_barrier_for_every_turn_is_not_enough():
    assert _orders(lambda tile: (0, tile % 2), 3) != set()
