"""The waits of the many-row 4-bit attention kernel as a model on the CPU: its roles are stepped in
random orders, some far slower than others, and no wait by parity may pass early or find its phase
gone.  The steps are those of ``csrc/fp4_attn_tile.cu``."""

import random

import pytest


class Barrier:
    """An mbarrier: a phase completes when ``count`` arrivals are in; waits see its parity only."""

    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passes(self, n):
        assert self.phase < n + 2, f"the wait for completion {n} finds {self.phase} of them: its phase is gone"
        if (self.phase ^ n) & 1:
            assert self.phase == n + 1, f"the wait for completion {n} passes at {self.phase}"
            return True
        return False


def _operands(bars, tiles):
    """An operand warp: K when S of the tile before is done, V of a window when the P V before is.
    ``tiles``: 0 for an ordinary tile, else the windows that its V takes."""
    n_pv = 0
    for n, windows in enumerate(tiles):
        if n > 0:
            yield "S", n - 1
        bars["K"].arrive()
        for _ in range(max(1, windows)):
            if n_pv > 0:
                yield "O", n_pv - 1
            bars["V"].arrive()
            n_pv += 1


def _softmax(bars, warp, tiles, meet):
    """A softmax warp; the first one issues the products (which complete at once).  A window is two
    products beside O, which every warp reads."""
    n_pv = n_p = n_t = 0
    for n, windows in enumerate(tiles):
        yield "K", n
        if meet:
            bars["ready"].arrive()
        if warp == 0:
            if meet:
                yield "ready", n
            if n_pv > 0:
                yield "O", n_pv - 1
            bars["S"].arrive()
        yield "S", n
        for _ in range(max(1, windows)):
            for half in range(2 if windows else 1):
                bars["P"].arrive()
                if warp == 0:
                    yield "V", n_pv
                    yield "P", n_p
                    if windows:
                        bars["T"].arrive()
                    if half == 1 or not windows:
                        bars["O"].arrive()
                n_p += 1
                if windows:
                    yield "T", n_t
                    n_t += 1
            n_pv += 1
    yield "O", n_pv - 1


def _run(seed, *, meet):
    rng = random.Random(seed)
    tiles = [rng.choice([0, 0, 0, 1, 3]) for _ in range(5)]
    bars = {name: Barrier(1 if name in "STO" else 4) for name in ("K", "V", "P", "S", "T", "O", "ready")}
    roles = [_operands(bars, tiles) for _ in range(4)] + [_softmax(bars, w, tiles, meet) for w in range(4)]
    speed = [rng.choice([1, 1, 100]) for _ in roles]
    waits = {i: next(r) for i, r in enumerate(roles)}
    while waits:
        able = [i for i, (name, n) in waits.items() if bars[name].passes(n)]
        assert able, f"nobody can go on: {waits}"
        i = rng.choices(able, [speed[i] for i in able])[0]
        try:
            waits[i] = next(roles[i])
        except StopIteration:
            del waits[i]


def test_no_wait_misses_its_phase():
    for seed in range(300):
        _run(seed, meet=True)


def test_the_model_finds_the_missing_meeting():
    """Where softmax warps do not meet before S is issued, one that is held up loses a phase of K."""
    with pytest.raises(AssertionError, match="phase is gone"):
        for seed in range(300):
            _run(seed, meet=False)


class Meeting:
    """A named barrier of four warps: a warp that arrives goes on when all four have."""

    def __init__(self):
        self.arrived, self.turns = 0, 0


def _operand_loop(meeting, words, warp, fails_at, tiles, agree):
    """An operand warp's turns, of which ``fails_at`` is the one where a wait of its runs out."""
    alive = True
    for n in range(tiles):
        if not agree and not alive:
            return
        words[warp] = not alive
        meeting.arrived += 1
        turn = meeting.turns
        if meeting.arrived == 4:
            meeting.arrived, meeting.turns = 0, meeting.turns + 1
            meeting.stop = any(words)
        while meeting.turns == turn:
            yield
        if agree and meeting.stop:
            return
        if fails_at == n:
            alive = False
        yield


def _ends(agree, late):
    meeting, words = Meeting(), [False] * 4
    roles = [_operand_loop(meeting, words, w, 2 if w == late else None, 6, agree) for w in range(4)]
    for _ in range(200):
        roles = [r for r in roles if next(r, "end") != "end"]
    return not roles


def test_operand_warps_end_together_when_a_wait_runs_out():
    """One warp's wait runs out and the others' do not: none is left at the named barrier."""
    assert all(_ends(True, late) for late in range(4))
    assert not any(_ends(False, late) for late in range(4))  # as it would be if each left alone
