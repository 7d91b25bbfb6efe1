"""The many-row attention kernel's roles as an event model, without a GPU.

Every role of csrc/kv_attn_tile.cu (copies, queries, a product warp per tile,
four softmax warps per tile) walks its units with its waits and arrivals in the
kernel's order; ring slots, blocks and arrival counts are the kernel's own
(csrc/kv_tile_order.h), durations are random and may differ from tile to tile.
A barrier tells the parity of its phase and nothing else, as on the GPU. A wait
for a phase is wrong when a later phase has completed by then (it would run out,
or be taken for a later one's), when an arrival comes that a phase has no room
for, when a ring slot changes under a product, and when nobody can go on.
"""
from __future__ import annotations

import ctypes as C
import heapq
import itertools
import random
import subprocess
from collections import defaultdict
from pathlib import Path

import pytest

from llm_shield_b200 import _build

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("order") / "libkv_tile_order.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", str(_build.CSRC),
                    str(HERE / "kv_tile_order.cpp"), "-o", str(out)], check=True)
    L = C.CDLL(str(out))
    L.order_new.restype = C.c_void_p
    L.order_new.argtypes = [C.c_int32, C.c_int32, C.c_int32, C.c_uint32]
    for name in ("order_delete", "order_ahead", "order_lead", "order_two", "order_block_step", "order_says_values_here"):
        getattr(L, name).argtypes = [C.c_void_p]
    for name in ("order_key_slot", "order_value_slot", "order_blocks_of", "order_first_block", "order_looker",
                 "order_frees_queries"):
        getattr(L, name).argtypes = [C.c_void_p, C.c_int32]
    return L


class Order:
    """One unit, by the kernel's header."""

    def __init__(self, L, nb, wide, clean, ring):
        h = L.order_new(nb, wide, clean, ring)
        tiles, blocks = range(2), range(nb)
        self.nb, self.wide, self.clean, self.ring = nb, bool(wide), clean, ring
        self.ahead, self.lead, self.two, self.step = L.order_ahead(h), L.order_lead(h), bool(L.order_two(h)), L.order_block_step(h)
        self.key_slot = [L.order_key_slot(h, b) for b in blocks]
        self.value_slot = [L.order_value_slot(h, b) for b in blocks]
        self.blocks_of = [L.order_blocks_of(h, a) for a in tiles]
        self.first = [L.order_first_block(h, a) for a in tiles]
        self.looker = [L.order_looker(h, a) for a in tiles]
        self.says_values_here = L.order_says_values_here(h)
        self.frees_queries = [L.order_frees_queries(h, a) for a in tiles]
        L.order_delete(h)


class Fault(Exception):
    pass


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.left, self.tx, self.phase, self.waiting = name, count, count, 0, 0, []


class Model:
    """speed[a]: how much longer tile a's softmax takes; grown[a]: how often its maxima grow."""

    def __init__(self, units, stages, rng, speed=(1.0, 1.0), grown=(0.1, 0.1), jitter=0.1, copy=700, rules=None, values_here=1, queries_free=3):
        self.units, self.stages, self.rng, self.speed, self.grown, self.jitter, self.copy = units, stages, rng, speed, grown, jitter, copy
        self.rules = rules or {}
        B = Barrier
        self.q_full, self.q_free = B("q_full", 1), B("q_free", queries_free)
        self.s_full = [[B(f"s_full {a} {h}", 1) for h in range(2)] for a in range(2)]
        self.p_full = [[B(f"p_full {a} {h}", 4) for h in range(2)] for a in range(2)]
        self.pv_done = [B(f"pv_done {a}", 1) for a in range(2)]
        self.o_full = [B(f"o_full {a}", 1) for a in range(2)]
        self.v_here = [B(f"v_here {a}", values_here) for a in range(2)]
        self.v_clean, self.join_ready = B("v_clean", 4), B("join_ready", 2)
        self.full = [B(f"full {s}", 1) for s in range(stages)]
        self.empty = [B(f"empty {s}", 2) for s in range(stages)]
        self.named = {1: [], 2: []}
        self.slot = [None] * stages
        self.now, self.tick, self.events, self.pipe = 0.0, itertools.count(), [], 0.0
        self.running = 0

    # ---- events
    def at(self, t, call):
        heapq.heappush(self.events, (t, next(self.tick), call))

    def took(self, mean):
        return mean * (1 + self.jitter * (2 * self.rng.random() - 1))

    def arrive(self, bar, n=1):
        if n == 0:
            return
        bar.left -= n
        if bar.left < 0:
            raise Fault(f"{bar.name}: more arrivals than a phase has")
        self.settle(bar)

    def settle(self, bar):
        if bar.left == 0 and bar.tx == 0:
            bar.phase += 1
            bar.left = bar.count
            woken, bar.waiting = bar.waiting, []
            for role, want in woken:
                self.at(self.now, lambda role=role, bar=bar, want=want: self.wait(role, bar, want))

    def expect(self, bar, nbytes):
        bar.tx += nbytes
        self.arrive(bar)

    def complete(self, bar, nbytes):
        bar.tx -= nbytes
        self.settle(bar)

    def wait(self, role, bar, want):
        """Phase number `want` of the barrier, of which the role only names the parity."""
        if bar.phase > want + 1:
            raise Fault(f"{bar.name}: phase {want} waited for when {bar.phase} were complete")
        if (bar.phase & 1) != (want & 1):
            if bar.phase != want + 1:
                raise Fault(f"{bar.name}: phase {want} taken for one of {bar.phase}")
            self.go(role)
        else:
            bar.waiting.append((role, want))

    def go(self, role):
        try:
            what = next(role)
        except StopIteration:
            self.running -= 1
            return
        if isinstance(what, tuple):
            self.wait(role, *what)
        elif isinstance(what, str):  # a named barrier of all eight softmax warps
            met = self.named[int(what)]
            met.append(role)
            if len(met) == 8:
                self.named[int(what)] = []
                for r in met:
                    self.at(self.now, lambda r=r: self.go(r))
        else:
            self.at(self.now + what, lambda: self.go(role))

    def product(self, cycles, slot, content, commits):
        """Queued behind what the tensor cores have; the commits' arrivals come when it is done."""
        if slot is not None and self.slot[slot % self.stages] != content:
            raise Fault(f"slot of {content} holds {self.slot[slot % self.stages]}")
        self.pipe = max(self.pipe, self.now) + cycles

        def done():
            if slot is not None and self.slot[slot % self.stages] != content:
                raise Fault(f"slot of {content} was overwritten")
            for bar, n in commits:
                for _ in range(n):
                    self.arrive(bar)
        self.at(self.pipe, done)

    # ---- roles
    def producer(self):
        for i, U in enumerate(self.units):
            def fill(slot, content):
                s = slot % self.stages
                yield self.empty[s], slot // self.stages - 1
                self.expect(self.full[s], 1)
                self.slot[s] = content
                self.at(self.now + self.took(self.copy), lambda: self.complete(self.full[s], 1))
            for b in range(U.ahead):
                yield from fill(U.key_slot[b], (i, "k", b))
            for b in range(U.nb):
                yield from fill(U.value_slot[b], (i, "v", b))
                if b + U.lead < U.nb:
                    yield from fill(U.key_slot[b + U.lead], (i, "k", b + U.lead))
                yield 20

    def queries(self):
        for i, U in enumerate(self.units):
            yield self.q_free, i - 1
            yield self.took(900)
            self.arrive(self.q_full)

    def products(self, a):
        done = cleaned = seen = 0
        for i, U in enumerate(self.units):
            n_blocks, b0 = U.blocks_of[a], U.first[a]
            frees = self.rules.get("frees_queries", lambda U, a: U.frees_queries[a])(U, a)

            def pass_to(slot):
                nonlocal seen
                while seen != slot:
                    s = seen % self.stages
                    yield self.full[s], seen // self.stages
                    self.arrive(self.empty[s])
                    seen += 1

            def filled(slot):
                nonlocal seen
                yield from pass_to(slot)
                seen += 1
                yield self.full[slot % self.stages], slot // self.stages

            def scores(n, h):
                b = b0 + n * U.step
                slot = U.key_slot[b]
                if h == 0:
                    yield from filled(slot)
                commits = [(self.s_full[a][h], 1)]
                if h == 1:
                    commits.append((self.empty[slot % self.stages], 1))
                    if n == n_blocks - 1:
                        commits.append((self.q_free, frees))
                self.product(256, slot, (i, "k", b), commits)
                yield 60

            def values(n, h):
                nonlocal cleaned
                b = b0 + n * U.step
                slot = U.value_slot[b]
                if h == 0:
                    yield from filled(slot)
                    if b >= U.clean:
                        says = self.rules.get("says_values_here", lambda U, a: U.says_values_here)(U, a)
                        self.arrive(self.v_here[U.looker[a]], says)
                        if U.wide and a == 1:
                            yield self.v_clean, cleaned
                            cleaned += 1
                yield self.p_full[a][h], done + n
                commits = [(self.pv_done[a], 1)]
                if h == 1:
                    commits.append((self.empty[slot % self.stages], 1))
                    if n == n_blocks - 1:
                        commits.append((self.o_full[a], 1))
                        if U.two:
                            commits.append((self.join_ready, 1))
                self.product(256, slot, (i, "v", b), commits)
                yield 60

            yield self.q_full, i
            if n_blocks:
                yield from scores(0, 0)
                yield from scores(0, 1)
            else:
                self.arrive(self.q_free, frees)
            for n in range(n_blocks):
                for h in range(2):
                    yield from values(n, h)
                    if n + 1 < n_blocks:
                        yield from scores(n + 1, h)
            yield from pass_to(U.ring + 2 * U.nb)
            done += n_blocks

    def softmax(self, a, w):
        done = ends = joins = looked = 0
        for U in self.units:
            n_blocks = U.blocks_of[a]
            for n in range(n_blocks):
                b = U.first[a] + n * U.step
                for h in range(2):
                    yield self.s_full[a][h], done + n
                    if h == 0 and b >= U.clean and U.looker[a] == a:
                        yield self.v_here[a], looked
                        looked += 1
                        yield self.took(150)
                        if U.wide:
                            self.arrive(self.v_clean)
                    if (n or h) and self.rng.random() < self.grown[a]:
                        yield self.pv_done[a], 2 * (done + n) + h - 1
                        yield self.took(400)
                    yield self.took(900) * self.speed[a]
                    self.arrive(self.p_full[a][h])
            if n_blocks:
                yield self.o_full[a], ends
            if U.two:
                if a == 1:
                    yield self.join_ready, joins
                    yield self.took(300)
                yield "1"
            if U.wide or a == 0:
                yield self.took(1500)
            done += n_blocks
            ends += n_blocks > 0
            joins += U.two
            if U.two:
                yield "2"
                if a == 0 and w == 0:
                    self.arrive(self.q_free)

    def run(self):
        roles = [self.producer(), self.queries(), self.products(0), self.products(1)]
        roles += [self.softmax(a, w) for a in range(2) for w in range(4)]
        self.running = len(roles)
        for r in roles:
            self.at(0.0, lambda r=r: self.go(r))
        while self.events:
            self.now, _, call = heapq.heappop(self.events)
            call()
        if self.running:
            raise Fault(f"{self.running} roles cannot go on")


def units_of(L, shapes):
    """(key blocks, two tiles?, masked blocks) in the order of one CTA."""
    out, ring = [], 0
    for nb, wide, masked in shapes:
        out.append(Order(L, nb, wide, max(nb - masked, 0), ring))
        ring += 2 * nb
    return out


def faults(L, shapes_of, stages, runs, rules=None, **kw):
    seen = defaultdict(int)
    for seed in range(runs):
        rng = random.Random(seed)
        counts = dict(values_here=L.values_here(), queries_free=L.queries_free())
        counts.update({k: v for k, v in (rules or {}).items() if k in counts})
        try:
            Model(units_of(L, shapes_of(rng)), stages, rng, rules=rules, **counts, **kw).run()
        except Fault as e:
            seen[str(e).split(":")[0]] += 1
    return dict(seen)


SPEEDS = [(1.0, 1.0), (1.0, 1.1), (1.0, 1.3), (1.0, 2.0), (1.3, 1.0), (2.0, 1.0), (1.0, 6.0), (6.0, 1.0)]


def two_tiles(rng):
    return [(rng.choice((1, 2, 3, 8, 16)), True, rng.randint(0, 4)) for _ in range(6)]


@pytest.mark.parametrize("stages", [4, 8])
@pytest.mark.parametrize("speed", SPEEDS, ids=str)
def test_units_of_two_tiles(lib, stages, speed):
    """Masked blocks one after another, one tile's softmax slower than the other's."""
    for kw in (dict(), dict(grown=(0.0, 1.0)), dict(grown=(1.0, 0.0), jitter=0.5), dict(copy=20)):
        assert faults(lib, two_tiles, stages, 12, speed=speed, **kw) == {}


def test_the_model_sees_a_look_that_runs_ahead(lib):
    """Values announced by tile 0 alone: its warpgroup may look through two blocks before tile 1 has waited for one."""
    rules = dict(says_values_here=lambda U, a: 0 if U.wide and a == 1 else 1, values_here=1)
    assert "v_clean" in faults(lib, two_tiles, 8, 20, rules=rules, speed=(1.0, 1.3))


def mixed(rng):
    return [rng.choice(((1, False, 1), (1, False, 0), (2, False, 1), (1, True, 1), (rng.randint(2, 9), rng.random() < 0.5, rng.randint(0, 3))))
            for _ in range(14)]


@pytest.mark.parametrize("stages", [4, 8])
@pytest.mark.parametrize("speed", SPEEDS, ids=str)
def test_units_of_one_tile_and_two(lib, stages, speed):
    """One-block units, which tile 1 has no block of, among others."""
    for kw in (dict(jitter=0.5), dict(grown=(0.0, 1.0)), dict(grown=(1.0, 0.0), jitter=0.5), dict(copy=20, jitter=0.9)):
        assert faults(lib, mixed, stages, 12, speed=speed, **kw) == {}


def test_the_model_sees_queries_that_run_ahead(lib):
    """A one-block unit's queries released by tile 0 alone: the next unit's may come before tile 1 has waited for these."""
    rules = dict(frees_queries=lambda U, a: (3 if a == 0 else 0) if U.nb == 1 and not U.wide else U.frees_queries[a])
    for stages in (4, 8):
        assert "q_full" in faults(lib, mixed, stages, 40, rules=rules, speed=(1.0, 2.0))


def test_ring_slots_are_taken_once_and_in_order(lib):
    for nb in range(1, 20):
        for wide in (0, 1):
            U = Order(lib, nb, wide, 0, 100)
            assert sorted(U.key_slot + U.value_slot) == list(range(100, 100 + 2 * nb))
            mine = [[U.first[a] + n * U.step for n in range(U.blocks_of[a])] for a in range(2)]
            assert (mine == [list(range(nb))] * 2) if wide else sorted(mine[0] + mine[1]) == list(range(nb))
            for a in range(2):  # each tile goes through the ring forwards
                walk = [slot for b in mine[a] for slot in (U.key_slot[b], U.value_slot[b])]
                assert walk == sorted(walk)
