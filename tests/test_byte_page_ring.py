"""The ring of byte pages in the attention over shared pages: a feeder copies pages into places, two warps take each of them, and behind the last page the feeder's arrival
at the next place tells them that there are no more.  Every interleaving is walked, with mbarriers as they are: a wait looks at the parity of a phase only, so a barrier
that goes on by two phases is missed by whoever waits for the first."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rexl3_b200", "ops", "csrc", "attention_shared.cu")


def stuck(pages: int, places: int, end_waits: bool):
    """-> None, or the state (full, empty, arrivals, feeder, takers) of an interleaving in which nobody can go on.  The end is signalled once both takers are past all
    pages but the last two: those the last product has waited for."""
    start = ((0,) * places, (0,) * places, (0,) * places, 0, (0, 0))      # phases completed of full and empty, arrivals at empty, pages copied (+ 1: ended), next page of each (-1: done)
    seen, stack = {start}, [start]
    passed = lambda phases, parity: phases & 1 != parity  # noqa: E731
    while stack:
        full, empty, arrived, fed, takers = state = stack.pop()
        after, at, turn = [], fed % places, fed // places
        if fed <= pages:
            free = turn == 0 or passed(empty[at], (turn - 1) & 1)
            ready = free if fed < pages or end_waits else True
            if fed == pages:
                ready = ready and all(t < 0 or t >= pages - 2 for t in takers)
            if ready:
                after.append((full[:at] + (full[at] + 1,) + full[at + 1:], empty, arrived, fed + 1, takers))
        for w in (0, 1):
            n = takers[w]
            if n < 0 or not passed(full[n % places], n // places & 1):
                continue
            if n >= pages:
                after.append((full, empty, arrived, fed, takers[:w] + (-1,) + takers[w + 1:]))
                continue
            p, count = n % places, arrived[n % places] + 1
            after.append((full, empty[:p] + (empty[p] + count // 2,) + empty[p + 1:], arrived[:p] + (count % 2,) + arrived[p + 1:], fed, takers[:w] + (n + 1,) + takers[w + 1:]))
        if not after and (fed <= pages or takers != (-1, -1)):
            return state
        for s in after:
            if s not in seen:
                seen.add(s)
                stack.append(s)
    return None


def end_waits_in_source() -> bool:
    text = open(SOURCE).read()
    end = re.search(r"ring_landed\(full, S, copied\);(.*?)mbar_arrive\(&full\[st\]\);", text, re.S).group(1)
    return re.search(r"round == 0 \|\| sh_wait\(&empty\[st\], \(round - 1\) & 1,", end) is not None


@pytest.mark.parametrize("pages", range(9))
def test_the_end_of_the_pages_reaches_both_warps(pages):
    assert stuck(pages, 2, end_waits_in_source()) is None


def test_an_end_that_does_not_wait_for_its_place_is_missed():
    assert stuck(1, 2, False) is None
    assert stuck(2, 2, False) is not None and stuck(7, 2, False) is not None
