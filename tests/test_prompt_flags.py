"""The V flags of the packed attention (csrc/vxk_prompt_attn.cu): the warps that look at V write an item's flag, the
softmax warps of its tiles A and B read it behind the item's last product.  A model of who waits for whom, on
the CPU, holds the slots to the furthest that the writers can get while a reader stands still."""
from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "voxtral.cpp_b200" / "csrc" / "vxk_prompt_attn.cu").read_text()
FLAGS = int(re.search(r"constexpr int kFlags = (\d+);", SOURCE).group(1))
STAGES = [int(n) for n in re.search(r"kStages = HD == 128 \? (\d+) : (\d+);", SOURCE).groups()]


def furthest_written(items, stages, s, k):
    """Last item that the V warps may have flagged while the warps of tile s have not read item k's flag.
    items: key tiles (A, B) of each."""
    # the issuer passes every item before the next one with a tile s, and of that one the scores alone
    held = next((i for i in range(k + 1, len(items)) if items[i][s]), None)
    if held is None:
        return len(items) - 1
    ring = sum(2 * max(n) for n in items[:held]) + 1  # tiles given back: all before, and the held item's first K
    reach, at = ring + stages, 0  # tiles [0, reach) may be in the ring or past it
    last = -1
    for i, n in enumerate(items):
        if at + 1 >= reach:  # its first V is tile at + 1
            break
        last = i
        at += 2 * max(n)
    return last


def overwritten(items, stages, slot):
    """Readers (item, tile) whose slot may hold a later item's flag."""
    found = []
    for s in (0, 1):
        for k in range(len(items)):
            if not items[k][s]:
                continue
            mine = slot(items, k, s)
            for i in range(k + 1, furthest_written(items, stages, s, k) + 1):
                if (items[i][s] or slot is by_item) and slot(items, i, s) == mine:
                    found.append((k, s))
                    break
    return found


def by_item(items, i, s):
    return i % FLAGS


def by_tile(items, i, s):
    return sum(1 for n in items[:i] if n[s]) % FLAGS


def _cases():
    rng = random.Random(1)
    yield [(1, 1)] + [(1, 0)] * 40 + [(1, 1)]
    yield [(1, 1)] * 60
    yield [(1, 0)] * 60
    for _ in range(200):
        lone = rng.random()
        yield [(n, 0) if rng.random() < lone else (n, n) for n in (rng.randint(1, 4) for _ in range(rng.randint(1, 80)))]


@pytest.mark.parametrize("stages", STAGES)
def test_flags_are_read_before_their_slot_is_written_again(stages):
    for items in _cases():
        assert overwritten(items, stages, by_tile) == []


@pytest.mark.parametrize("stages", STAGES)
def test_the_model_finds_slots_by_item_unsafe(stages):
    assert (0, 1) in overwritten([(1, 1)] + [(1, 0)] * 40 + [(1, 1)], stages, by_item)


def test_the_kernel_counts_items_by_tile():
    assert "nth[s] % kFlags" in SOURCE and SOURCE.count("nth % kFlags") == 2 and "(i - begin) % kFlags" not in SOURCE
