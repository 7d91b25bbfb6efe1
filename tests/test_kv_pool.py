"""Host bookkeeping of the paged cache without a GPU: page numbers, counts,
moves and refusals against a plain model, and every attention plan's pieces
against the (token, key) pairs they have to cover, each once and in bounds."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

from llm_shield_b200 import _build, binding

HERE = Path(__file__).resolve().parent
FEW_TILE = 16


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv") / "libkv_host.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror",
                    "-I", str(_build.CSRC), "-I", str(_build.INCLUDE), str(HERE / "kv_host.cpp"), "-o", str(out)], check=True)
    L = C.CDLL(str(out))
    P, I, J = C.c_void_p, C.c_int32, C.c_int64
    L.host_new.restype, L.host_new.argtypes = P, [I, I]
    L.host_delete.argtypes = [P]
    L.host_error.restype, L.host_error.argtypes = C.c_char_p, [P]
    L.host_open.argtypes = [P, I, P]
    L.host_extend.argtypes = [P, P, P, I]
    L.host_fork.argtypes = [P, P, P, I, I, P]
    L.host_free.argtypes = [P, P, I]
    L.host_compact.argtypes = L.host_used.argtypes = L.host_spanned.argtypes = [P]
    L.host_moves.argtypes = [P, P]
    L.host_len.argtypes = [P, J]
    L.host_pages.argtypes = [P, J, P]
    L.host_plan.argtypes = [P, P, P, I, I, I, I, J, J, J, J, I]
    L.host_plan_array.argtypes, L.host_plan_array.restype = [P, I, P], J
    L.host_part_rows.argtypes, L.host_part_rows.restype = [P], J
    return L


class HostPool:
    def __init__(self, L, pages, pt):
        self.L, self.h, self.pt, self.n_pages = L, C.c_void_p(L.host_new(pages, pt)), pt, pages

    def __del__(self):
        self.L.host_delete(self.h)

    @staticmethod
    def _a(x, t):
        return np.ascontiguousarray(x, t)

    def check(self, rc):
        if rc:
            raise binding.ShieldError(rc, self.L.host_error(self.h).decode())

    def open(self, n):
        out = np.empty(n, np.int64)
        self.check(self.L.host_open(self.h, n, out.ctypes.data))
        return out

    def extend(self, ids, counts):
        i, c = self._a(ids, np.int64), self._a(counts, np.int32)
        self.check(self.L.host_extend(self.h, i.ctypes.data, c.ctypes.data, i.size))

    def fork(self, ids, lens=None, share=True):
        i = self._a(ids, np.int64)
        l = None if lens is None else self._a(lens, np.int32)
        out = np.empty(i.size, np.int64)
        self.check(self.L.host_fork(self.h, i.ctypes.data, None if l is None else l.ctypes.data, i.size, int(share), out.ctypes.data))
        return out

    def free(self, ids):
        i = self._a(ids, np.int64)
        self.check(self.L.host_free(self.h, i.ctypes.data, i.size))

    def compact(self):
        self.check(self.L.host_compact(self.h))
        return self.moves()

    def moves(self):
        out = np.empty((self.L.host_moves(self.h, None), 3), np.int32)
        self.L.host_moves(self.h, out.ctypes.data)
        return out

    def pages(self, i):
        out = np.empty(self.L.host_pages(self.h, int(i), None), np.int32)
        self.L.host_pages(self.h, int(i), out.ctypes.data)
        return out.tolist()

    def length(self, i):
        return self.L.host_len(self.h, int(i))

    def plan(self, ids, counts, group=4, kv_heads=2, few_rows=FEW_TILE, items=1 << 20, segs=None, part=1 << 24, table=1 << 24, mode=0):
        i, c = self._a(ids, np.int64), self._a(counts, np.int32)
        rc = self.L.host_plan(self.h, i.ctypes.data, c.ctypes.data, i.size, group, kv_heads, few_rows, items,
                              2 * i.size if segs is None else segs, part, table, mode)
        if rc < 0:
            return None
        self.check(rc)
        get = {}
        for k, (name, width) in enumerate([("slot", 1), ("perm", 1), ("lim", 1), ("merge", 3), ("segs", 8), ("few", 8),
                                           ("tile", 8), ("where", 1), ("table", 1)]):
            a = np.empty(self.L.host_plan_array(self.h, k, None), np.int32)
            self.L.host_plan_array(self.h, k, a.ctypes.data)
            get[name] = a if width == 1 else a.reshape(-1, width)
        get["part_rows"] = self.L.host_part_rows(self.h)
        return get


class Model:
    """The same pool in plain Python: what each page holds, by position."""

    def __init__(self, pages, pt):
        self.pt, self.n = pt, pages
        self.seqs = {}
        self.content = {}  # (page, row) -> (token that was written there)

    def held(self):
        return {p for l, pages in self.seqs.values() for p in pages}

    def take(self):
        p = min(set(range(self.n)) - self.held() - self.busy)
        self.busy.add(p)
        return p

    def extend(self, ids, counts):
        self.busy = set()
        for i, c in zip(ids, counts):
            l, pages = self.seqs[i]
            for p in range(l, l + c):
                if p // self.pt >= len(pages):
                    pages.append(self.take())
                self.content[pages[p // self.pt], p % self.pt] = (i, p)
            self.seqs[i] = (l + c, pages)

    def apply(self, moves):
        old = dict(self.content)
        for src, dst, rows in moves:
            for r in range(rows):
                self.content[dst, r] = old[src, r]

    def read(self, i):
        l, pages = self.seqs[i]
        return [self.content[pages[p // self.pt], p % self.pt] for p in range(l)]


@pytest.mark.parametrize("seed", range(12))
def test_pool_against_a_plain_model(host, seed):
    rng = random.Random(seed)
    pt = rng.choice((16, 32))
    n_pages = rng.choice((9, 70, 150))
    H, M = HostPool(host, n_pages, pt), Model(n_pages, pt)
    said = {}  # what each sequence has to read back
    for step in range(120):
        live = list(M.seqs)
        op = rng.choice(("open", "extend", "extend", "fork", "copy", "free", "compact"))
        try:
            if op == "open":
                for i in H.open(rng.randint(1, 3)).tolist():
                    M.seqs[i], said[i] = (0, []), []
            elif op == "extend" and live:
                ids = rng.sample(live, rng.randint(1, min(4, len(live))))
                counts = [rng.randint(0, 3 * pt) for _ in ids]
                H.extend(ids, counts)
                M.extend(ids, counts)
                for i in ids:
                    said[i] = said[i] + [(i, p) for p in range(len(said[i]), M.seqs[i][0])]
            elif op in ("fork", "copy") and live:
                ids = [rng.choice(live) for _ in range(rng.randint(1, 4))]
                lens = [rng.randint(0, M.seqs[i][0]) for i in ids] if rng.random() < 0.5 else None
                kids = H.fork(ids, lens, share=op == "fork").tolist()
                moves = H.moves().tolist()
                M.busy = set()
                want = []
                for k, (i, kid) in enumerate(zip(ids, kids)):
                    l = M.seqs[i][0] if lens is None else lens[k]
                    pages = []
                    for j in range(-(-l // pt)):
                        if op == "fork" and (j + 1) * pt <= l:
                            pages.append(M.seqs[i][1][j])
                        else:
                            pages.append(M.take())
                            want.append([M.seqs[i][1][j], pages[-1], min(pt, l - j * pt)])
                    M.seqs[kid] = (l, pages)
                    said[kid] = said[i][:l]
                assert moves == want
                M.apply(moves)
            elif op == "free" and live:
                ids = rng.sample(live, rng.randint(1, len(live)))
                H.free(ids)
                for i in ids:
                    del M.seqs[i], said[i]
            elif op == "compact":
                moves = H.compact().tolist()
                held, used = M.held(), len(M.held())
                assert [m[0] for m in moves] == sorted((p for p in held if p >= used), reverse=True)
                assert [m[1] for m in moves] == sorted(p for p in range(used) if p not in held)
                M.apply(moves)
                to = {m[0]: m[1] for m in moves}
                M.seqs = {i: (l, [to.get(p, p) for p in pages]) for i, (l, pages) in M.seqs.items()}
                assert host.host_spanned(H.h) == used
        except binding.ShieldError as e:
            assert e.code == binding.ERR_NOMEM and op in ("extend", "fork", "copy")
        for i, (l, pages) in M.seqs.items():
            assert H.length(i) == l and H.pages(i) == pages
            assert M.read(i) == said[i]
        assert host.host_used(H.h) == len(M.held())


def test_refusals_change_nothing(host):
    H = HostPool(host, 4, 16)
    a, b = H.open(2).tolist()
    H.extend([a, b], [20, 16])
    before = [(H.length(i), H.pages(i)) for i in (a, b)]
    for call, code in [
        (lambda: H.extend([a, a], [1, 1]), binding.ERR_ARG),
        (lambda: H.extend([a, b], [1, -1]), binding.ERR_RANGE),
        (lambda: H.extend([a, 99], [1, 1]), binding.ERR_ARG),
        (lambda: H.extend([a, b], [12, 17]), binding.ERR_NOMEM),
        (lambda: H.extend([a], [2**31 - 1 - 20]), binding.ERR_RANGE),
        (lambda: H.fork([a, a]), binding.ERR_NOMEM),
        (lambda: H.fork([a], [21]), binding.ERR_RANGE),
        (lambda: H.fork([a], [-1]), binding.ERR_RANGE),
        (lambda: H.fork([b, b], share=False), binding.ERR_NOMEM),
        (lambda: H.free([a, b, a]), binding.ERR_ARG),
        (lambda: H.free([a, 12345]), binding.ERR_ARG),
    ]:
        with pytest.raises(binding.ShieldError) as e:
            call()
        assert e.value.code == code
        assert [(H.length(i), H.pages(i)) for i in (a, b)] == before and host.host_used(H.h) == 3
    H.extend([a, b], [0, 0])
    assert host.host_used(H.h) == 3
    H.free([a])  # an ended sequence's id does not name the next one in its place
    (c,) = H.open(1).tolist()
    assert c != a
    with pytest.raises(binding.ShieldError):
        H.extend([a], [1])
    H.extend([c], [1])


def check_plan(H, ids, counts, P, group, kv_heads):
    """Every visible (token, head row, key) exactly once, through addresses inside the sequence's own pages."""
    pt = H.pt
    start = np.concatenate([[0], np.cumsum(counts)])
    T = int(start[-1])
    owner = np.repeat(np.arange(len(ids)), counts)
    pages = [H.pages(i) for i in ids]
    lens = [H.length(i) for i in ids]
    pos = np.array([lens[s] - counts[s] + t - start[s] for t, s in enumerate(owner)], np.int64)
    assert P["slot"].tolist() == [pages[s][p // pt] * pt + p % pt for s, p in zip(owner, pos)]
    assert sorted(P["perm"].tolist()) == list(range(T))
    assert (P["lim"] == pos[P["perm"]] + 1).all()
    seen = [np.zeros((group, p + 1), np.int8) for p in pos]  # per token in batch order
    part_used = np.zeros(P["part_rows"], np.int8)
    segs = P["segs"].tolist()
    of_part = {}  # first partial row -> (segment, split, tile)
    for s, (tok0, rows, slot0, ntiles, nsplit, tile_rows, parent, direct) in enumerate(segs):
        assert parent < s and ntiles == -(-rows // tile_rows) and (not direct or (parent == -1 and nsplit == 1))
        for sp in range(nsplit):
            for t in range(ntiles):
                w = int(P["where"][slot0 + sp * ntiles + t])
                if w >= 0:
                    assert w not in of_part and not direct
                    of_part[w] = (s, sp, t)
    inside = {}  # token in plan order -> segments whose pieces hold its rows
    for kind, name in ((0, "few"), (1, "tile")):
        cost = None
        for it in P[name].tolist():
            tok0, r0, nr, k0, k1, table, part, masked = it
            assert 1 <= nr <= (FEW_TILE if kind == 0 else 256)
            assert 0 <= k0 < k1 and k0 % pt == 0
            keys = (k1 - k0) * (2 if nr > 128 else 1)
            assert cost is None or keys <= cost  # longest first
            cost = keys
            if part >= 0:
                s, sp, t = of_part.pop(part)
                assert segs[s][0] == tok0 and r0 == t * segs[s][5] and nr == min(segs[s][5], segs[s][1] - r0)
                rows = part_used[part:part + nr * kv_heads]
                assert rows.size == nr * kv_heads and not rows.any()
                rows[:] = 1
                for t in range(tok0 + r0 // group, tok0 + (r0 + nr - 1) // group + 1):
                    inside.setdefault(t, set()).add(s)
            first = int(P["lim"][tok0 + r0 // group])
            for r in range(r0, r0 + nr):
                tok = int(P["perm"][tok0 + r // group])
                lim = int(P["lim"][tok0 + r // group])
                assert lim >= first or not masked  # masks start behind the first row's
                if not masked:
                    assert lim >= k1
                own = pages[owner[tok]]
                last = (min(lim, k1) - 1) // pt + 1
                if lim > k0:
                    assert P["table"][table + k0 // pt:table + last].tolist() == own[k0 // pt:last]
                assert table + (k1 - 1) // pt < P["table"].size
                row = seen[tok][r % group]
                assert not row[k0:min(k1, lim)].any()
                row[k0:min(k1, lim)] = 1
    assert part_used.all() and not of_part
    for tok in range(T):
        assert seen[tok].all()
    joined = P["merge"].tolist()
    assert [t for t, _, _ in joined] == sorted(inside)
    for t, token, leaf in joined:  # every piece that holds a joined token's rows is on its way to the root
        assert token == P["perm"][t]
        chain, s = set(), leaf
        while s >= 0:
            assert 0 <= t - segs[s][0] < segs[s][1] // group
            chain.add(s)
            s = segs[s][6]
        assert inside[t] <= chain


def tree(H, rng, depth, width, lo, hi):
    level = H.open(rng.randint(1, 2)).tolist()
    H.extend(level, [rng.randint(lo, hi) for _ in level])
    for _ in range(depth):
        kids = []
        for i in level:
            n = H.length(i)
            ids = [i] * rng.randint(1, width)
            kids += H.fork(ids, [n if rng.random() < 0.6 else rng.randint(0, n) for _ in ids]).tolist()
        H.extend(kids, [rng.randint(0 if rng.random() < 0.3 else 1, hi) for _ in kids])
        level = kids
    return level


@pytest.mark.parametrize("seed", range(24))
@pytest.mark.parametrize("few_rows", [0, FEW_TILE, 2**31 - 1])
def test_plans_cover_every_pair_once(host, seed, few_rows):
    rng = random.Random(seed)
    H = HostPool(host, 20000, rng.choice((16, 64, 128)))
    ids = tree(H, rng, rng.randint(0, 3), rng.randint(1, 5), 1, rng.choice((40, 900, 3000)))
    rng.shuffle(ids)
    ids = ids[:24]
    top = rng.choice((1, 6, 300))
    counts = [min(H.length(i), rng.randint(0, top)) for i in ids]
    group, kv_heads = rng.choice(((1, 3), (4, 2), (7, 1), (20, 1)))
    for mode in (0, 1, 2, 3):
        P = H.plan(ids, counts, group, kv_heads, few_rows, mode=mode)
        check_plan(H, ids, counts, P, group, kv_heads)


def test_shared_prefix_is_one_segment(host):
    H = HostPool(host, 4000, 64)
    (root,) = H.open(1).tolist()
    H.extend([root], [2048 + 17])
    kids = H.fork([root] * 40).tolist()
    H.extend(kids, [5] * 40)
    P = H.plan(kids, [1] * 40, group=4, kv_heads=8)
    top = [s for s in P["segs"].tolist() if s[6] == -1]
    assert len(top) == 1 and top[0][5] >= 128 and len(P["segs"]) == 41
    keys = {(it[3], it[4]) for it in P["tile"].tolist()}
    assert min(k[0] for k in keys) == 0 and max(k[1] for k in keys) == 2048
    # a token inside the shared pages keeps its own causal limit: nothing behind it is shared
    early = H.fork([root] * 3, [100, 100, 100]).tolist()
    P = H.plan(early, [70, 1, 100])
    check_plan(H, early, [70, 1, 100], P, 4, 2)


def test_small_capacities_fall_back_or_refuse(host):
    H = HostPool(host, 4000, 64)
    (root,) = H.open(1).tolist()
    H.extend([root], [4096])
    kids = H.fork([root] * 8).tolist()
    H.extend(kids, [3] * 8)
    for part in (0, 100, 5000):
        P = H.plan(kids, [3] * 8, part=part)
        assert P["part_rows"] <= part
        check_plan(H, kids, [3] * 8, P, 4, 2)
    with pytest.raises(binding.ShieldError):
        H.plan(kids, [3] * 8, table=10)
    empty = H.plan([], [])
    assert not empty["few"].size and not empty["tile"].size
    assert not H.plan(kids, [0] * 8)["perm"].size


def test_long_runs_are_cut_into_many_pieces(host):
    H = HostPool(host, 2000, 64)
    (root,) = H.open(1).tolist()
    H.extend([root], [60000])
    P = H.plan([root], [1], group=8, kv_heads=1)
    assert P["segs"][0][4] > 32
    check_plan(H, [root], [1], P, 8, 1)


@pytest.mark.parametrize("pt", [16, 128])
def test_a_planned_compaction_changes_nothing_until_it_is_taken(host, pt):
    rng = random.Random(pt)
    host.host_plan_compact.argtypes = [C.c_void_p]
    p = HostPool(host, 300, pt)
    ids = list(p.open(30))
    p.extend(ids, [rng.randint(0, 6 * pt) for _ in ids])
    ids += list(p.fork(ids[:10]))
    gone = rng.sample(ids, 15)
    p.free(gone)
    live = [i for i in ids if i not in gone]

    def state():
        return [(p.length(i), p.pages(i)) for i in live], host.host_used(p.h), host.host_spanned(p.h)

    before = state()
    for _ in range(2):
        p.check(host.host_plan_compact(p.h))
        assert state() == before
    p.extend(live[:1], [1])  # pages are handed out as before the plan
    held = {x for i in live for x in p.pages(i)}
    p.check(host.host_plan_compact(p.h))
    planned = p.moves()
    np.testing.assert_array_equal(p.compact(), planned)
    assert len(planned) and host.host_spanned(p.h) == host.host_used(p.h) == len(held)


def test_capacities_grow_a_few_times(host):
    rng = random.Random(0)
    for most in (1, 7, 512, 8192, 2 ** 31 - 1):
        have = times = 0
        for need in range(1, min(most, 20000) + 1):
            now = host.host_grown(have, need, most)
            assert need <= now <= max(most, need) and now >= have
            times += now != have
            have = now
        assert times <= 16
        for _ in range(200):
            have, need = rng.randint(0, most), rng.randint(1, most)
            assert max(have, need) <= host.host_grown(have, need, most) <= most


def test_steps_that_meet_on_a_page(host):
    """Against the slots of the plan: a meeting is a slot that appears twice."""
    host.host_steps_meet.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32]
    rng, seen = random.Random(5), set()
    for _ in range(150):
        p = HostPool(host, 400, 16)
        ids = list(p.open(3))
        p.extend(ids, [rng.randint(0, 70) for _ in ids])
        for _ in range(2):
            ids += list(p.fork(rng.choices(ids, k=3)))
            p.extend(ids, [rng.choice((0, 0, 1, 16, 20)) for _ in ids])
        batch = rng.sample(ids, rng.randint(1, 6))
        counts = [min(p.length(i), rng.choice((0, 1, 5, 16, 40))) for i in batch]
        slots = p.plan(batch, counts)["slot"]
        twice = len(set(slots.tolist())) < len(slots)
        i, c = np.asarray(batch, np.int64), np.asarray(counts, np.int32)
        assert bool(host.host_steps_meet(p.h, i.ctypes.data, c.ctypes.data, len(batch))) == twice
        seen.add(twice)
    assert seen == {True, False}


def test_an_id_is_never_given_twice(host):
    """Past the turns that an id counts, a slot is left alone and the next one is taken."""
    host.host_churn.argtypes, host.host_churn.restype = [C.c_void_p, C.c_int64], C.c_int64
    p = HostPool(host, 8, 16)
    (first,) = p.open(1)
    p.free([first])
    assert host.host_churn(p.h, (1 << 22) + 5) == 0  # pairs of open and free that gave an id of an earlier one again
    (now,) = p.open(1)
    assert now != first
    with pytest.raises(binding.ShieldError):
        p.extend([first], [1])
    p.extend([now], [3])
    assert host.host_used(p.h) == 1 and host.host_sequences(p.h) == 1
    p.free([now])
    assert host.host_used(p.h) == 0 and host.host_sequences(p.h) == 0
