"""The order of the prompt kernel's roles over the quantised cache (csrc/kv_quant_attn_tc.cu), from its barriers: what one role
leaves in shared memory for another, in rings indexed by the tile, is read before the next tile that has the slot overwrites it."""
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "emberlm_b200" / "csrc" / "kv_quant_attn_tc.cu"


def ring():
    return int(re.search(r"constexpr int kRing = (\d+);", SOURCE.read_text()).group(1))


class Order:
    """Events (role, tile) of `tiles` tiles and what each one waits for."""

    def __init__(self, tiles):
        self.before = {}
        self.tiles = tiles
        for g in range(tiles):
            # warp 0: the stage's codes and scales must have been converted two tiles ago; keys and values in turn
            self.edge(("load k", g), ("make k", g - 2), ("load v", g - 1))
            self.edge(("load v", g), ("make v", g - 2), ("load k", g))
            # warp 2: keys and values in turn
            self.edge(("look k", g), ("load k", g), ("look v", g - 1))
            self.edge(("look v", g), ("load v", g), ("look k", g))
            # converting warps: their stage is free once the product that read it has finished
            self.edge(("make k", g), ("look k", g), ("S", g - 2), ("make k", g - 1))
            self.edge(("make v", g), ("look v", g), ("PV", g - 2), ("make v", g - 1))
            # warp 1: S(0), S(1), then PV(j) and S(j + 2) in turn; S waits for the values' looks too
            self.edge(("issue S", g), ("make k", g), ("look v", g), ("issue PV", g - 2), ("issue S", g - 1))
            self.edge(("issue PV", g), ("make v", g), ("softmax", g), ("issue S", g + 1))
            self.edge(("S", g), ("issue S", g))
            self.edge(("PV", g), ("issue PV", g))
            # the softmax warps read what was left for the tile, then arrive
            self.edge(("softmax", g), ("S", g), ("softmax", g - 1))

    def edge(self, event, *needs):
        self.before[event] = [n for n in needs if 0 <= n[1] < self.tiles]

    def ordered(self, first, then):
        """Whether `first` has happened whenever `then` does."""
        seen, todo = set(), [then]
        while todo:
            for e in self.before[todo.pop()]:
                if e == first:
                    return True
                if e not in seen:
                    seen.add(e)
                    todo.append(e)
        return False


@pytest.mark.parametrize("reader,writer", [
    ("softmax", "look k"),      # scale_k
    ("softmax", "look v"),      # shrink_o, exp_v, the marks of NaN
    ("make k", "look k"),       # exp_k
    ("make v", "look v"),       # exp_v
    ("issue S", "look v"),      # a phase of the barriers `told`, which the issuer must not miss
])
def test_a_slot_of_the_ring_is_read_before_it_is_written_again(reader, writer):
    tiles, n = 40, ring()
    order = Order(tiles)
    for g in range(tiles - n):
        assert order.ordered((reader, g), (writer, g + n)), (reader, writer, g)
