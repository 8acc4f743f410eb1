"""The recurrence kernels' way of passing a state from tile to tile, as a small model run under random interleavings: blocks
take tiles from a counter, publish a tile's pair, look back for the nearest state behind words that are all set, fold
forward, publish the state.  Whatever the interleaving, every block finishes, and every state has the bits of the plain
sequential fold."""

from __future__ import annotations

import random

import numpy as np
import pytest

RESET = np.float32(-1)


def fold(pair, h):
    """``h <- A h + B`` as one fused operation; a pair marked A < 0 stands for a state."""
    a, b = pair
    return b if a < 0 else np.float32(np.float64(a) * np.float64(h) + np.float64(b))


def block(tile, chain, words, window):
    """One block's steps; yields between any two accesses another block could come between.  ``window`` words are seen one
    after the other, so a word may change while the later ones are read."""
    pair = chain[tile]
    yield
    words[tile] = pair
    yield
    if tile == 0:
        h = np.float32(0)
    else:
        while True:
            seen = []
            for back in range(window):
                seen.append(words[tile - 1 - back] if tile - 1 - back >= 0 else (RESET, np.float32(0)))
                yield
            unset = next((k for k, w in enumerate(seen) if w is None), window)
            state = next((k for k, w in enumerate(seen) if w is not None and w[0] < 0), window)
            if state < unset:
                break
        h = np.float32(0)
        for k in range(state, -1, -1):
            h = fold(seen[k], h)
    if not pair[0] < 0:
        words[tile] = (RESET, fold(pair, h))
    yield
    return


def run(chains, resident, window, rng):
    words = [[None] * len(c) for c in chains]
    order = [(t, c) for t in range(len(chains[0])) for c in range(len(chains))]  # time first, as the counter gives them
    order.reverse()
    live, steps = [], 0
    while order or live:
        while order and len(live) < resident:
            tile, c = order.pop()
            live.append(block(tile, chains[c], words[c], window))
        at = rng.randrange(len(live)) if rng.random() < 0.9 else len(live) - 1  # the youngest one often gets ahead
        try:
            next(live[at])
        except StopIteration:
            live.pop(at)
        steps += 1
        assert steps < 2_000_000, "the blocks wait for one another for good"
    return words


@pytest.mark.parametrize("chains,tiles,resident,window", [(1, 40, 1, 4), (1, 40, 12, 12), (3, 25, 7, 4), (8, 12, 20, 4), (2, 30, 64, 48)])
def test_every_interleaving_gives_the_sequential_bits(chains, tiles, resident, window):
    rng = random.Random(chains * 1000 + resident)
    data = []
    for _ in range(chains):
        pairs = []
        for t in range(tiles):
            a, b = np.float32(rng.uniform(0.2, 1.0)), np.float32(rng.gauss(0, 1))
            pairs.append((RESET, b) if t == 0 or rng.random() < 0.1 else (a, b))  # a sequence starts here and there
        data.append(pairs)
    want = []
    for pairs in data:
        h, states = np.float32(0), []
        for p in pairs:
            h = fold(p, h)
            states.append(h)
        want.append(states)
    for _ in range(12):
        words = run(data, resident, window, rng)
        for states, got in zip(want, words):
            assert all(w[0] < 0 for w in got)
            assert [w[1].tobytes() for w in got] == [s.tobytes() for s in states]
