"""The products of the attention kernels wait for the rows behind a sequence's end to be overwritten with zeros; only pieces
that have such rows do.  A wait asks for a phase by its parity, so it may also be answered by the phase two turns earlier,
unless something that was waited for before tells that that one is over.  Every interleaving of the loads' warp, the zeros'
warp and the products' warp, with the waits that the source has."""
import re
from pathlib import Path

import pytest

import configurable_hierarchical_allreduce_algorithms_b200 as chb

SOURCE = (Path(chb.__file__).parent / "csrc" / "kernels" / "attention.cu").read_text()
# the operand in the ring of two slots, the one in the ring of three (forward: the tile's keys, a ring of two that the zeros'
# warp has nothing to do with), and the zeros' barrier
KERNELS = {"attn_forward": ("vfull", "kfull", "vready"), "attn_dq": ("vfull", "kfull", "ready"), "attn_dkv": ("gfull", "qfull", "ready")}


def products_waits(kernel):
    """Barriers that the products' warp waits for ahead of the first product that may read the tile's zeros, in their order:
    (with zeros, without)."""
    body = SOURCE[SOURCE.index(f"{kernel}(const __grid_constant__"):]
    two, three, zeros = KERNELS[kernel]
    if kernel == "attn_forward":
        text = body[body.index("const auto scores"):body.index("mma_ts(")]
        waits = re.findall(r"bar_wait_warp\((\w+) \+ 8 \* s, \(g >> 1\)", text)
        assert re.search(rf"!ragged \|\| bar_wait_warp\({zeros}", text) or "values" in waits
        return [zeros] if "values" in waits else waits, [two]
    text = body[body.index("const auto scores"):body.index("const auto dprobs")]
    if re.search(rf"ragged \? {zeros} \+", text):
        return [zeros], [three]
    a, b = re.search(r"ragged \? (.*?)\n?\s+: (bar_wait_warp.*?)\)\) return", text, re.S).groups()
    return re.findall(r"bar_wait_warp\((\w+)", a), re.findall(r"bar_wait_warp\((\w+)", b)


def first_early_product(kernel, waits_ragged, waits_plain, ragged):
    """``ragged``: for every tile whether its piece waits for the zeros.  The first tile whose product could run before the
    zeros are there, over all interleavings; None: never."""
    two, three, zeros = KERNELS[kernel]
    ring = {two: 2, three: 2 if kernel == "attn_forward" else 3, zeros: 2}
    n = len(ragged)
    # (loads of `two`, loads of `three`, turns of the zeros' warp, products): each warp's turns come in order
    todo, seen = [(0, 0, 0, 0)], set()
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        a, b, z, m = state
        done = {two: a, three: b, zeros: z}

        def passes(bar, use):
            # turns of this slot that are over; a wait by parity passes on that many, and on two fewer than are asked for
            over = len(range(use % ring[bar], done[bar], ring[bar]))
            return (over - (use // ring[bar] + 1)) % 2 == 0

        free3 = m if kernel == "attn_forward" else min(m, z)
        if a < n and a - 2 < min(m, z):
            todo.append((a + 1, b, z, m))
        if b < n and b - ring[three] < free3:
            todo.append((a, b + 1, z, m))
        if z < n and z < a and (kernel == "attn_forward" or z < b):
            todo.append((a, b, z + 1, m))
        if m < n and all(passes(w, m) for w in (waits_ragged if ragged[m] else waits_plain)):
            if ragged[m] and z <= m:
                return m
            # (a plain tile's other operand is waited for too, ahead of the product that reads it)
            if ragged[m] or (m < a and m < b):
                todo.append((a, b, z, m + 1))
    return None


PATTERNS = [[False] * 5 + [True] * 4, [True, False, False, False, True, True, False, False, True], [False, True] * 5, [True] * 7]


@pytest.mark.parametrize("kernel", KERNELS)
def test_products_come_behind_the_zeros(kernel):
    waits = products_waits(kernel)
    for ragged in PATTERNS:
        assert first_early_product(kernel, *waits, ragged) is None


@pytest.mark.parametrize("kernel", KERNELS)
def test_the_zeros_alone_would_not_do(kernel):
    two, three, zeros = KERNELS[kernel]
    plain = [two] if kernel == "attn_forward" else [three]
    assert first_early_product(kernel, [zeros], plain, PATTERNS[0]) is not None
    if kernel != "attn_forward":      # (nor the ring of three: its load may come a turn ahead of the zeros' last one)
        assert first_early_product(kernel, [three, zeros], plain, PATTERNS[0]) is not None
