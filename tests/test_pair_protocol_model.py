"""Model check of how the pairs of gn_linear4.cu give up and end (CPU, no CUDA).

A pair's two loaders, the thread that multiplies and the warps that take the sums are restated step by step, with barriers of phases,
copies and products that land in their own time, and waits that may run out anywhere; the rules by which a warp takes
its turns and the pair ends are compiled from csrc/gn_turns.h.  Checked under many random interleavings:
  * a tile's result is its own complete sums, or NaN: never old or half-done sums, and nothing overwrites sums that are still being read;
  * when a CTA ends, no copy into its memory and no arrival at its barriers is under way;
  * every run ends, and one in which no wait runs out has all results.
Each `yield` is one access to a barrier or to memory, so the scheduler can switch threads between any two.
"""
import ctypes
import os
import random
import subprocess

import pytest

from channels_last_groupnorm_b200 import build

STAGES, WARPS = 2, 2


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    folder = tmp_path_factory.mktemp("turns")
    source, lib = folder / "turns.cpp", folder / "turns.so"
    source.write_text("""#include "gn_turns.h"
using namespace gnb200;
extern "C" {
int take(int gone, int there, int* now_gone) { Turns t; t.gone = gone; const bool whole = t.take(there); *now_gone = t.gone; return whole; }
int missing(int k, int own, int peers) { return missing_of(k, own, peers); }
int begin(int own, int stages) { return drain_begin(own, stages); }
int end(int own, int peers) { return drain_end(own, peers); }
}
""")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", build.CSRC, str(source), "-o", str(lib)])
    return ctypes.CDLL(os.fspath(lib))


class Bar:
    """An mbarrier: a phase ends when all arrivals are there and as many bytes as were announced."""

    def __init__(self, count):
        self.count = self.pending = count
        self.bytes = self.phase = 0

    def _turn(self):
        if self.pending == 0 and self.bytes == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def arrive(self, announced=0):
        assert self.pending > 0, "an arrival that no phase has room for"
        self.bytes += announced
        self.pending -= 1
        self._turn()

    def landed(self, n):
        self.bytes -= n
        self._turn()

    def there(self, parity):
        return (self.phase & 1) != parity


class Pair:
    def __init__(self, seed, tiles, ktiles, giving_up, rules, turns="new", ends="new"):
        self.rng, self.tiles, self.ktiles, self.giving_up, self.rules = random.Random(seed), tiles, ktiles, giving_up, rules
        self.old_turns, self.old_ends = turns == "old", ends == "old"
        # full: the leader's, of both CTAs' copies; empty, sums, last: one each; taken: the leader's
        self.full, self.taken = [Bar(1) for _ in range(STAGES)], Bar(2 * WARPS)
        self.empty, self.sums, self.last = [[Bar(1) for _ in range(STAGES)] for _ in range(2)], [Bar(1), Bar(1)], [Bar(1), Bar(1)]
        self.gave_up, self.loads, self.multiplied, self.announced = [False, False], [0, 0], 0, 0
        self.copies, self.arrivals, self.queue = [], [], []  # under way: CTAs of copies; (CTA, barrier); products and commits, in order
        self.stage = [[None] * STAGES for _ in range(2)]
        self.acc, self.out, self.left = None, {}, [0, 0]
        self.met = [0, 0, 0]
        self.ended = [False, False]

    # waits: limited as in the kernels
    def wait(self, cta, bar, parity, checks=True):
        """producer_wait / consumer_wait: True where the phase is there"""
        while not bar.there(parity):
            if checks and self.gave_up[cta]:
                return bar.there(parity)
            if self.giving_up and self.rng.random() < self.giving_up:
                self.gave_up[cta] = True
                return bar.there(parity)
            yield
        return True

    def until(self, bar, parity):
        """a wait at the end: has to come by itself"""
        while not bar.there(parity):
            yield

    def barrier(self, which, everyone):
        self.met[which] += 1
        while self.met[which] < everyone:
            yield

    def loader(self, cta):
        n = 0
        for t in range(self.tiles):
            for k in range(self.ktiles):
                s = n % STAGES
                if n >= STAGES:
                    yield from self.wait(cta, self.empty[cta][s], (n // STAGES - 1) & 1)
                    if self.gave_up[cta]:
                        self.loads[cta] = n
                        return
                if cta == 0:
                    self.full[s].arrive(2)
                yield
                self.copies.append((cta, s, (t, k)))
                n += 1
                yield
        if not self.old_ends:
            for k in range(self.rules.begin(n, STAGES), n):
                yield from self.wait(cta, self.empty[cta][k % STAGES], (k // STAGES) & 1)
        self.loads[cta] = n

    def product(self):
        n = 0
        for t in range(self.tiles):
            for k in range(self.ktiles):
                s = n % STAGES
                yield from self.wait(0, self.full[s], (n // STAGES) & 1)
                if self.gave_up[0]:
                    break
                if k == 0 and t > 0:
                    yield from self.wait(0, self.taken, (t - 1) & 1)
                    if self.gave_up[0]:
                        break
                self.queue.append(("product", s, (t, k)))
                self.queue.append(("commit", [(c, self.empty[c][s]) for c in (0, 1)]))
                n += 1
                self.multiplied = n
                yield
            else:
                self.announced += 1
                self.queue.append(("commit", [(c, self.sums[c]) for c in (0, 1)]))
                yield
                continue
            break
        self.queue.append(("commit", [(0, self.last[0])]))
        yield from self.until(self.last[0], 0)

    def taker(self, cta, warp):
        gone = ctypes.c_int(0)
        for t in range(self.tiles):
            whole = False
            if self.old_turns or not gone.value:
                whole = yield from self.wait(cta, self.sums[cta], t & 1)
            if not self.old_turns:
                whole = bool(self.rules.take(gone.value, whole, ctypes.byref(gone)))
            yield
            read = self.acc if whole else "NaN"
            self.out[cta, warp, t] = read
            yield
            if whole or self.old_turns:
                self.taken.arrive()
            yield

    def thread(self, cta, body, leads):
        """A thread from its work to the pair's end; leads: it is the CTA's thread 0"""
        yield from body
        self.left[cta] += 1
        everyone = WARPS + 1 + (cta == 0)
        while self.left[cta] < everyone:
            yield
        if leads and self.old_ends and cta == 0:  # the leader's loader: its own copies, as far as it got
            for k in range(max(0, self.loads[0] - STAGES), self.loads[0]):
                for _ in range(20):
                    if self.full[k % STAGES].there((k // STAGES) & 1):
                        break
                    yield
        yield from self.barrier(0, 2 * WARPS + 3)
        if not self.old_ends:
            if any(self.gave_up):
                yield from self.barrier(1, 2 * WARPS + 3)
                if leads:
                    for k in range(self.rules.begin(self.multiplied, STAGES), self.multiplied):
                        yield from self.until(self.empty[cta][k % STAGES], (k // STAGES) & 1)
                    if self.announced:
                        yield from self.until(self.sums[cta], (self.announced - 1) & 1)
                    own, peers = self.loads
                    for k in range(self.rules.begin(own, STAGES), self.rules.end(own, peers) if cta == 0 else 0):
                        missing = self.rules.missing(k, own, peers)
                        if missing == 1:
                            self.full[k % STAGES].arrive(1)
                        elif missing == 2:
                            self.full[k % STAGES].landed(1)
                        yield from self.until(self.full[k % STAGES], (k // STAGES) & 1)
                yield from self.barrier(2, 2 * WARPS + 3)
        self.left[cta] += 1
        if self.left[cta] == 2 * everyone:
            self.ended[cta] = True
            assert not [c for c in self.copies if c[0] == cta], "a copy into a CTA that has ended"
            assert not [a for a in self.arrivals if a[0] == cta], "an arrival at a CTA that has ended"
            assert not [1 for q in self.queue if q[0] == "product"], "products of a pair that has ended"
            assert not [1 for q in self.queue if q[0] == "commit" and any(c == cta for c, _ in q[1])], "an arrival to come at a CTA that has ended"

    def land(self):
        """something that is under way takes its effect"""
        kinds = [kind for kind, some in (("copy", self.copies), ("arrival", self.arrivals), ("queue", self.queue)) if some]
        if not kinds:
            return False
        kind = self.rng.choice(kinds)
        if kind == "copy":
            cta, s, what = self.copies.pop(self.rng.randrange(len(self.copies)))
            self.stage[cta][s] = what
            self.full[s].landed(1)
        elif kind == "arrival":
            self.arrivals.pop(self.rng.randrange(len(self.arrivals)))[1].arrive()
        else:
            first = self.queue.pop(0)
            if first[0] == "product":
                _, s, what = first
                assert self.stage[0][s] == self.stage[1][s] == what, "a product of the wrong stage"
                self.acc = what if what[1] < self.ktiles - 1 else (what[0], "whole")
            else:
                self.arrivals += first[1]
        return True

    def run(self):
        threads = []
        for cta in (0, 1):
            threads += [self.thread(cta, self.taker(cta, w), w == 0) for w in range(WARPS)] + [self.thread(cta, self.loader(cta), False)]
        threads.append(self.thread(0, self.product(), False))
        idle, pace = 0, self.rng.choice([0.5, 0.3, 0.05])
        while threads:
            idle += 1
            assert idle < 60000, "does not end"
            if self.rng.random() < pace:
                self.land()
            t = self.rng.choice(threads)
            try:
                next(t)
            except StopIteration:
                threads.remove(t)
        for (cta, warp, t), got in self.out.items():
            assert got == "NaN" or got == (t, "whole"), "tile %d has %s" % (t, got)
        return sum(got != "NaN" for got in self.out.values()), any(self.gave_up)


SIZES = [(1, 1), (1, 5), (2, 1), (3, 1), (3, 3), (5, 2)]


@pytest.mark.parametrize("tiles,ktiles", SIZES)
def test_nothing_runs_out(rules, tiles, ktiles):
    for seed in range(100):
        results, gave_up = Pair(seed, tiles, ktiles, 0.0, rules).run()
        assert results == 2 * WARPS * tiles and not gave_up


@pytest.mark.parametrize("tiles,ktiles", SIZES)
@pytest.mark.parametrize("chance", [0.3, 0.05, 0.01])
def test_waits_run_out(rules, tiles, ktiles, chance):
    some = sum(Pair(seed, tiles, ktiles, chance, rules).run()[1] for seed in range(200))
    assert some  # (there were runs that gave up)


@pytest.mark.parametrize("old,words", [({"turns": "old"}, "has|room"), ({"ends": "old"}, "has ended")])
def test_the_model_sees_what_the_rules_are_for(rules, old, words):
    """Without them it finds results of other sums, and copies or arrivals behind a CTA's end."""
    found = set()
    for seed in range(300):
        tiles, ktiles = SIZES[seed % len(SIZES)]
        try:
            Pair(seed, tiles, ktiles, 0.05, rules, **old).run()
        except AssertionError as e:
            found.add(str(e).split("\n")[0])
    assert any(w in f for f in found for w in words.split("|")), found
