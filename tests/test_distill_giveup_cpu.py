"""Waits that give up in the persistent distillation kernel (sdmchat_b200/csrc/distill.cu, distill_rows_kernel), played
through on the host thread by thread.  Any wait that is not satisfied may run out, in one thread of a team and not in
another.  Whatever runs out, every thread has to come to its end (a team's barriers wait without limit, so its threads
leave together or not at all), no copy may still be under way into the block's shared memory when the last of
them has ended, and a row that is finished has been read whole.  Threads that leave each for itself do not keep to that."""
import random

import pytest

BUFFERS, RING, TEAMS, THREADS = 3, 6, 2, 3


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0, "more arrivals than a phase has"
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def done(self, parity):
        return self.phase & 1 != parity


class Meeting:
    """A team's barrier with an and over what its threads bring."""

    def __init__(self):
        self.here, self.round, self.said, self.all = 0, 0, True, True

    def enter(self, ok):
        self.here, self.said = self.here + 1, self.said and ok
        if self.here == THREADS:
            self.all, self.here, self.said, self.round = self.said, 0, True, self.round + 1


def play(rows, weights, rnd, run_out, together):
    """run_out: the chance, a look, that a wait gives up.  Returns the rows that each thread finished."""
    full, empty = [Barrier(2) for _ in range(RING)], [Barrier(THREADS) for _ in range(RING)]
    buffer, flying, finished = [None] * BUFFERS, {}, {}

    def wait(bar, parity):
        while not bar.done(parity):
            if rnd.random() < run_out:
                return False
            yield "wait"
        return True

    def loader(p):
        i = p
        while i < rows:
            last = i - BUFFERS
            if last >= 0 and not (yield from wait(empty[last % RING], last // RING & 1)):
                if not together:
                    yield from wait(full[last % RING], last // RING & 1)
                    return
                break
            assert buffer[i % BUFFERS] is None or buffer[i % BUFFERS][1] == last
            buffer[i % BUFFERS] = ("loading", i)
            flying[i] = rnd.choice([0, 1, 5, 60])
            for _ in range(rnd.randint(0, 3)):
                yield "work"
            full[i % RING].arrive()  # the teacher is there; the copy arrives when it lands
            yield "work"
            i += TEAMS
        if together:
            for u in range(1, RING // TEAMS + 1):
                j = i - u * TEAMS
                if j >= 0:
                    while not full[j % RING].done(j // RING & 1):
                        yield "wait"

    def copies():
        while running - {me_copies}:
            for i in list(flying):
                flying[i] -= 1
                if flying[i] < 0:
                    del flying[i]
                    buffer[i % BUFFERS] = ("whole", i)
                    full[i % RING].arrive()
            yield "work" if flying else "wait"

    def thread(t, me, meet):
        here = True
        for i in range(t, rows, TEAMS):
            if together:
                here = here and (yield from wait(full[i % RING], i // RING & 1))
            elif not (yield from wait(full[i % RING], i // RING & 1)):
                yield from wait(full[i % RING], i // RING & 1)
                return
            if weights[i]:
                for step in range(3):  # the first barrier of a row tells
                    mine = meet.round
                    meet.enter(here)
                    while meet.round == mine:
                        yield "meet"
                    if step == 0 and not meet.all:
                        return
                    assert buffer[i % BUFFERS] == ("whole", i)
            finished[i] = finished.get(i, 0) + 1
            if here:
                empty[i % RING].arrive()
            yield "work"

    tasks, running = {}, set()
    for p in range(TEAMS):
        tasks["loader", p] = loader(p)
        meet = Meeting()
        for me in range(THREADS):
            tasks["thread", p, me] = thread(p, me, meet)
    me_copies = "copies"
    tasks[me_copies] = copies()
    running.update(tasks)
    idle = 0
    while running - {me_copies}:
        name = rnd.choice(sorted(running, key=str))
        try:
            did = next(tasks[name])
        except StopIteration:
            running.discard(name)
            did = "work"
        idle = idle + 1 if did != "work" else 0
        if idle > 4000 and run_out > 0:
            raise AssertionError("threads wait at a barrier that nobody else comes to")
        assert idle < 100000
    assert not flying, "a copy is under way into a block that has ended"
    return finished


def weights_of(rows, seed):
    w = random.Random(seed)
    return [w.random() < (0.9, 0.5, 0.1)[seed % 3] for _ in range(rows)]


def test_without_a_timeout_every_row_is_finished():
    for seed in range(60):
        assert play(40, weights_of(40, seed), random.Random(seed), 0.0, True) == {i: THREADS for i in range(40)}


def test_threads_that_give_up_leave_together():
    short = 0
    for seed in range(400):
        done = play(40, weights_of(40, seed), random.Random(seed), (0.3, 0.05, 0.005)[seed % 3], True)
        short += len(done) < 40
    assert short > 100  # waits did run out


def test_threads_that_leave_each_for_itself_do_not_end():
    with pytest.raises(AssertionError):
        for seed in range(400):
            play(40, weights_of(40, seed), random.Random(seed), (0.3, 0.05, 0.005)[seed % 3], False)
