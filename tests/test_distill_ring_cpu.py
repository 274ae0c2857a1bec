"""The barrier protocol of the persistent distillation kernel (sdmchat_b200/csrc/distill.cu, distill_rows_kernel), played
through on the host under random schedules: two warps load rows into three buffers, two teams take the rows in turn, and
a wait sees of a barrier only the parity of its phase.  With barriers by rows mod 6 every row is loaded into a free
buffer and read when it is whole; barriers by buffer (mod 3) would let a wait mistake a phase for the one two before it."""
import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0, "more arrivals than a phase has"
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def done(self, parity):  # what mbarrier.try_wait.parity sees
        return self.phase & 1 != parity


def play(rows, ring, rnd):
    full, empty, buffer = [Barrier(2) for _ in range(ring)], [Barrier(1) for _ in range(ring)], [None] * 3

    def loader(p):
        for i in range(p, rows, 2):
            last = i - 3
            while last >= 0 and not empty[last % ring].done(last // ring & 1):
                yield
            assert buffer[i % 3] is None
            buffer[i % 3] = ("loading", i)
            full[i % ring].arrive()
            for _ in range(rnd.randint(0, 5)):
                yield
            buffer[i % 3] = ("whole", i)
            full[i % ring].arrive()
            yield

    def team(t):
        for i in range(t, rows, 2):
            while not full[i % ring].done(i // ring & 1):
                yield
            assert buffer[i % 3] == ("whole", i)
            for _ in range(rnd.choice([0, 0, 20])):  # a row of weight 0 takes no time
                yield
            buffer[i % 3] = None
            empty[i % ring].arrive()
            yield

    running = [loader(0), loader(1), team(0), team(1)]
    for _ in range(200000):
        if not running:
            return
        one = rnd.choice(running)
        try:
            next(one)
        except StopIteration:
            running.remove(one)
    raise AssertionError("the schedule does not end")


def test_six_barriers_keep_rows_and_phases_apart():
    for seed in range(100):
        play(60, 6, random.Random(seed))


def test_three_barriers_would_not():
    with pytest.raises(AssertionError):
        for seed in range(20):
            play(60, 3, random.Random(seed))
