"""Rings whose slots are waited for by parity: which rings several consumers may take in turn.

A wait for filling number n of a slot (counted from 0) passes when the slot's count of completed fillings has not the
parity of n: for n + 1 completed, as meant, but also for n - 1.  A consumer that took filling n - 1 itself never sees that
count; one that takes every other item of a ring with an odd number of slots took n - 2, and may."""
import itertools
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "blackwell-inference-server_b200" / "csrc"


def _stale_reads(slots, items, arrivals, consumers=2):
    """Items that a consumer would take before they are there: consumers take the items in turn, each as soon as its wait
    passes; the producer fills a slot when its last item has been taken; item i arrives at arrivals[i] or later."""
    count, taken, issued, at = [0] * slots, set(), {}, 0
    heads, stale = list(range(consumers)), []
    landed = set()
    for now in itertools.count():
        while at < items and (at < slots or at - slots in taken):
            issued[at] = now
            at += 1
        for i, t in issued.items():
            if i not in landed and now >= max(t, arrivals[i]):
                landed.add(i)
                count[i % slots] += 1
        for c in range(consumers):
            i = heads[c]
            if i < items and count[i % slots] % 2 != (i // slots) % 2:
                if i not in landed:
                    stale.append(i)
                    return stale
                taken.add(i)
                heads[c] += consumers
        if all(h >= items for h in heads):
            return stale


@pytest.mark.parametrize("slots", [4, 5, 6, 7, 8, 9])
def test_which_rings_two_consumers_may_share(slots):
    items = 4 * slots
    late = [_stale_reads(slots, items, [0 if i != slow else 10**3 for i in range(items)]) for slow in range(items - 1)]
    if slots % 2:
        assert any(late), "an odd ring gives an item that is not there to the other consumer"
    else:
        assert not any(late)


@pytest.mark.parametrize("slots,safe", [(3, True), (4, False), (6, True)])
def test_three_consumers(slots, safe):
    items = 4 * slots * 3
    late = [_stale_reads(slots, items, [0 if i != slow else 10**3 for i in range(items)], 3) for slow in range(items - 1)]
    assert any(late) != safe


def test_the_merge_sees_every_filling():
    """Three groups take the tiles of four W slots: the MMA thread, which takes all, waits for a tile's W before the
    commit that the tile's group waits for."""
    text = (CSRC / "lora.cu").read_text()
    issuer = text[text.index("umma_commit(&aempty[sa]);"):text.index("umma_commit(&dfull[db]);")]
    assert "mbar_wait(&wfull[i % SW], (i / SW) & 1" in issuer


def test_the_requantiser_has_an_even_ring():
    text = (CSRC / "lora.cu").read_text()
    assert re.search(r"pl\.stages = std::min\(kReqMaxStages, .*\) / 2 \* 2;", text)
    assert int(re.search(r"kReqMaxStages = (\d+)", text)[1]) % 2 == 0


def test_the_gemm_asserts_it():
    text = (CSRC / "gemm.cu").read_text()
    assert re.search(r"static_assert\(STAGES % 2 == 0 && ASTAGES % 2 == 0 && XSTAGES % NI == 0", text)
