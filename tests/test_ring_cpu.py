"""The ring of operand stages of the 32-bit product (csrc/linear.cu), as a model: one warp requests copies in order, which arrive in any order; teams take the
stages in turn and prepare them; one warp uses them up in order.  Barriers are asked by parity: the answer to "is the phase of parity p over?" is
whether the phase that is open now has the other one."""
import random

import pytest


class Ring:
    def __init__(self, rng, stages, teams, blocks, waits):
        self.rng, self.S, self.T, self.n, self.waits = rng, stages, teams, blocks, waits
        self.full, self.split, self.empty = [0] * stages, [0] * stages, [0] * stages  # phases that are over
        self.in_flight, self.holds = [], [None] * stages                              # copies, what a stage's bytes are
        self.load, self.use = 0, 0
        self.next = list(range(teams))                                                # each team's k-block
        self.seen = [0] * teams                                                       # how many of its waits for that are over
        self.wrong = False

    @staticmethod
    def over(phases, parity):
        return phases & 1 != parity

    def question(self, st, wait):
        bar, parity = wait
        return (self.full if bar == "full" else self.empty)[st], parity

    def step(self):
        """One of the things that can happen happens; False when there is none."""
        able = []
        if self.load < self.n:
            st, ph = self.load % self.S, self.load // self.S & 1
            if self.load < self.S or self.over(self.empty[st], ph ^ 1):
                able.append(("load", st))
        able += [("arrive", i) for i in range(len(self.in_flight))]
        for t in range(self.T):
            if self.next[t] < self.n:
                st, ph = self.next[t] % self.S, self.next[t] // self.S & 1
                if self.over(*self.question(st, self.waits(ph)[self.seen[t]])):
                    able.append(("team", t))
        if self.use < self.n and self.over(self.split[self.use % self.S], self.use // self.S & 1):
            able.append(("use", self.use % self.S))
        if not able:
            return False
        what, i = self.rng.choice(able)
        if what == "load":
            self.in_flight.append((self.load, i))
            self.load += 1
        elif what == "arrive":
            block, st = self.in_flight.pop(i)
            self.holds[st] = block
            self.full[st] += 1
        elif what == "team":
            self.seen[i] += 1
            if self.seen[i] == len(self.waits(0)):
                st = self.next[i] % self.S
                self.wrong |= self.holds[st] != self.next[i]
                self.split[st] += 1
                self.next[i] += self.T
                self.seen[i] = 0
        else:
            self.wrong |= self.holds[i] != self.use
            self.empty[i] += 1
            self.use += 1
        return True

    def run(self):
        while not self.wrong and self.step():
            pass
        return not self.wrong and self.use == self.n


def used_up_then_full(ph):
    return ("empty", ph ^ 1), ("full", ph)


def full_only(ph):
    return (("full", ph),)


def both_copies(ph):
    return ("full", ph ^ 1), ("full", ph)


@pytest.mark.parametrize("stages", [3, 4, 7, 8])
def test_teams_that_wait_for_the_last_round_to_be_used_up_take_no_stage_too_early_and_do_not_hang(stages):
    rng = random.Random(stages)
    assert all(Ring(rng, stages, 3, 40, used_up_then_full).run() for _ in range(1500))


@pytest.mark.parametrize("stages", [4, 7, 8])
@pytest.mark.parametrize("waits", [full_only, both_copies])
def test_the_model_sees_what_other_waits_do(stages, waits):
    """The copy's barrier alone lets a team pass too early; asked for the copy before as well, it hangs when both have arrived."""
    rng = random.Random(stages)
    assert not all(Ring(rng, stages, 3, 40, waits).run() for _ in range(1500))


def test_the_copys_barrier_is_enough_where_a_stage_has_one_team():
    rng = random.Random(1)
    assert all(Ring(rng, 6, 3, 40, full_only).run() for _ in range(500))
