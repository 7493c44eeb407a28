"""The paged cache's bookkeeping and the attention plan on the CPU.

The C++ that the library uses for both has no device code; it is compiled here
with the host compiler and followed step by step by a model of a few lines: a
dictionary of sequences whose tokens carry distinct labels, and a pool of
labelled slots.  A plan is checked by what it must do: give every row each of
its sequence's positions exactly once, through the right pages.
"""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OK, BAD_SEQ, REPEATED, BAD_COUNT, NO_PAGES, NO_SEQS = range(6)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv_host") / "kv_host.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D_GLIBCXX_ASSERTIONS", "-Wall", "-Wextra", "-shared", "-fPIC",
                    "-I", os.path.join(HERE, "..", "edgexpu-llm_amd", "csrc"), os.path.join(HERE, "kv_host.cpp"), "-o",
                    so], check=True)
    L = C.CDLL(so)
    L.host_new.restype = C.c_void_p
    for f in ("host_free", "host_seq", "host_fork", "host_extend", "host_truncate", "host_release", "host_compact",
              "host_free_pages", "host_moves", "host_len", "host_pages", "host_plan", "host_plan_get"):
        n = {"host_fork": 4, "host_extend": 3, "host_truncate": 2, "host_release": 2, "host_moves": 1, "host_len": 1,
             "host_pages": 2, "host_plan": 8, "host_plan_get": 2}.get(f, 0)
        getattr(L, f).argtypes = [C.c_void_p] + [C.c_void_p if (f, i) in _POINTERS else C.c_int for i in range(n)]
    return L


_POINTERS = {("host_fork", 1), ("host_fork", 3), ("host_extend", 1), ("host_extend", 2), ("host_release", 1),
             ("host_moves", 0), ("host_pages", 1), ("host_plan", 1), ("host_plan", 2), ("host_plan", 5), ("host_plan_get", 1)}


def ints(v):
    return (C.c_int * max(1, len(v)))(*v)


class Host:
    """The compiled bookkeeping beside a pool of labels that follows its copies."""

    def __init__(self, lib, page, n_pages, max_seqs):
        self.L, self.page, self.n_pages, self.max_seqs = lib, page, n_pages, max_seqs
        self.h = lib.host_new(page, n_pages, max_seqs)
        self.pool = np.zeros((n_pages, page), np.int64)
        self.want = {}  # sequence -> its tokens' labels
        self.next = 1

    def __del__(self):
        self.L.host_free(self.h)

    def moves(self):
        n = self.L.host_moves(self.h, None)
        a = np.zeros((n, 3), np.int32)
        if n:
            self.L.host_moves(self.h, a.ctypes.data)
        # all at once on the device: no page is both read and written, none written twice
        assert len(set(a[:, 1])) == n and not set(a[:, 0]) & set(a[:, 1])
        for s, d, u in a:
            assert 0 < u <= self.page
            self.pool[d, :u] = self.pool[s, :u]
        return n

    def pages(self, s):
        n = self.L.host_pages(self.h, s, None)
        a = np.zeros(n, np.int32)
        if n:
            self.L.host_pages(self.h, s, a.ctypes.data)
        return a

    def new(self):
        s = self.L.host_seq(self.h)
        free = [i for i in range(self.max_seqs) if i not in self.want]
        assert s == (free[0] if free else -1)
        if s >= 0:
            self.want[s] = []
        return s

    def extend(self, seqs, n_new):
        st = self.L.host_extend(self.h, len(seqs), ints(seqs), ints(n_new))
        if st != OK:
            return st
        self.moves()
        for s, n in zip(seqs, n_new):
            p = self.pages(s)
            for _ in range(n):
                i = len(self.want[s])
                self.pool[p[i // self.page], i % self.page] = self.next
                self.want[s].append(self.next)
                self.next += 1
        return OK

    def fork(self, parents, copy):
        out = (C.c_int * max(1, len(parents)))()
        st = self.L.host_fork(self.h, len(parents), ints(parents), copy, out)
        if st != OK:
            return st, []
        assert (self.moves() > 0) == (copy and any(len(self.want[p]) for p in parents))
        for p, c in zip(parents, out):
            assert c not in self.want
            self.want[c] = list(self.want[p])
        return OK, list(out)[: len(parents)]

    def check(self):
        used = {}
        for s, labels in self.want.items():
            assert self.L.host_len(self.h, s) == len(labels)
            p = self.pages(s)
            assert len(p) == -(-len(labels) // self.page)
            got = self.pool[p].reshape(-1)[: len(labels)]
            assert list(got) == labels, f"sequence {s} reads other tokens than its own"
            for i in p:
                used.setdefault(int(i), set()).add(s)
            assert len(set(p)) == len(p)
        assert self.L.host_free_pages(self.h) == self.n_pages - len(used)
        return used


@pytest.mark.parametrize("seed", range(12))
def test_random_histories(lib, seed):
    r = random.Random(seed)
    page = r.choice([16, 32, 64])
    h = Host(lib, page, r.choice([7, 64, 65, 130]), r.choice([3, 20]))
    refused = 0
    for _ in range(400):
        live = sorted(h.want)
        op = r.choice(["new", "extend", "extend", "extend", "fork", "truncate", "release", "compact"])
        if op == "new":
            h.new()
        elif op == "extend" and live:
            ids = r.sample(live, r.randint(1, len(live)))
            before = {s: list(h.pages(s)) for s in live}
            st = h.extend(ids, [r.choice([0, 1, r.randint(0, 3 * page)]) for _ in ids])
            assert st in (OK, NO_PAGES)
            if st == NO_PAGES:
                refused += 1
                assert before == {s: list(h.pages(s)) for s in live}
        elif op == "fork" and live:
            ids = [r.choice(live) for _ in range(r.randint(1, 3))]
            st, _ = h.fork(ids, r.random() < 0.3)
            assert st in (OK, NO_PAGES, NO_SEQS)
        elif op == "truncate" and live:
            s = r.choice(live)
            n = r.randint(0, len(h.want[s]))
            assert h.L.host_truncate(h.h, s, n) == OK
            del h.want[s][n:]
        elif op == "release" and live:
            ids = r.sample(live, r.randint(1, max(1, len(live) // 3)))
            assert h.L.host_release(h.h, len(ids), ints(ids)) == OK
            for s in ids:
                del h.want[s]
        elif op == "compact":
            n = h.L.host_compact(h.h)
            h.moves()
            used = h.check()
            assert n == len(used) and sorted(used) == list(range(n))
        h.check()
    assert h.next > 50


def test_lowest_pages_first(lib):
    h = Host(lib, 16, 200, 4)
    a, b = h.new(), h.new()
    h.extend([a], [16 * 70])
    h.extend([b], [16 * 3])
    assert list(h.pages(a)) == list(range(70)) and list(h.pages(b)) == [70, 71, 72]
    h.L.host_truncate(h.h, a, 16 * 2 + 1)
    del h.want[a][33:]
    h.extend([b], [16 * 2])
    assert list(h.pages(b)) == [70, 71, 72, 3, 4]
    h.check()


def test_last_holder_grows_in_place(lib):
    h = Host(lib, 32, 20, 5)
    a = h.new()
    h.extend([a], [40])
    _, (b,) = h.fork([a], 0)
    shared = h.pages(a)[-1]
    # both grow in one call: the first gets a copy, the other is alone by then
    assert h.extend([a, b], [1, 1]) == OK
    assert h.pages(a)[-1] != shared and h.pages(b)[-1] == shared and h.pages(a)[0] == h.pages(b)[0]
    h.check()
    # a whole last page is shared without a copy
    c = h.new()
    h.extend([c], [32])
    _, (d,) = h.fork([c], 0)
    h.extend([d], [1])
    assert h.L.host_moves(h.h, None) == 0 and h.pages(c)[0] == h.pages(d)[0]


def test_refusals_change_nothing(lib):
    h = Host(lib, 16, 4, 3)
    a, b = h.new(), h.new()
    assert h.extend([a], [33]) == OK
    assert h.extend([a, a], [1, 1]) == REPEATED
    assert h.extend([b, 2], [1, 1]) == BAD_SEQ and h.extend([-1], [1]) == BAD_SEQ and h.extend([99], [1]) == BAD_SEQ
    assert h.extend([a], [-1]) == BAD_COUNT
    assert h.extend([a, b], [1, 17]) == NO_PAGES
    assert h.extend([b], [2**31 - 1]) == NO_PAGES
    assert h.L.host_truncate(h.h, a, 34) == BAD_COUNT and h.L.host_truncate(h.h, a, -1) == BAD_COUNT
    assert h.L.host_truncate(h.h, 2, 0) == BAD_SEQ
    assert h.L.host_release(h.h, 2, ints([a, a])) == REPEATED and h.L.host_release(h.h, 1, ints([2])) == BAD_SEQ
    assert h.fork([a], 1)[0] == NO_PAGES
    st, (c,) = h.fork([a], 0)
    assert st == OK and h.fork([a], 0)[0] == NO_SEQS
    # the page that a copy on write needs counts too: 3 pages held, 1 free
    assert h.extend([b], [16]) == OK
    assert h.extend([a], [1]) == NO_PAGES
    h.check()
    assert h.L.host_release(h.h, 1, ints([c])) == OK
    del h.want[c]
    assert h.extend([a], [1]) == OK
    h.check()


# ------------------------------------------------------------------ the plan


def plan(h, seqs, n_new, group, n_kv=2, cost=(47, 56, 59, 83), part_cost=104, wgs=512):
    h.L.host_plan(h.h, len(seqs), ints(seqs), ints(n_new), group, n_kv, ints(cost), part_cost, wgs)
    out = []
    for what, w in enumerate((4, 8, 1, 1, 1, 1, 2)):
        n = h.L.host_plan_get(h.h, what, None)
        a = np.zeros(max(n, 1), np.int32)
        h.L.host_plan_get(h.h, what, a.ctypes.data)
        out.append(a[:n].reshape(-1, w) if w > 1 else a[:n])
    return out


def check_plan(h, seqs, n_new, group, **kw):
    tokens, items, pages, join_rows, join_at, join_parts, ((parts, writable),) = plan(h, seqs, n_new, group, **kw)
    flat = [(s, len(h.want[s]) - n + i) for s, n in zip(seqs, n_new) for i in range(n)]
    assert [tuple(t[:2]) for t in tokens] == [(p, h.pages(s)[p // h.page] * h.page + p % h.page) for s, p in flat]
    assert sorted(tokens[:, 2]) == list(range(len(flat)))
    assert all(tokens[t[2], 0] == t[3] for t in tokens)
    seen = [[] for _ in range(len(flat) * group)]
    row_parts = [[] for _ in seen]
    next_part = 0
    for row0, n_rows, key0, key1, at, causal, part, _ in items:
        assert 0 < n_rows <= 128 and key0 < key1 and key0 % 16 == 0
        next_part += n_rows if part >= 0 else 0
        for r in range(row0, row0 + n_rows):
            t = tokens[r // group]
            hi = min(key1, t[3] + 1) if causal else key1
            assert causal or key1 <= t[3], "a shared run reaches the row's own tokens"
            seen[r] += [(p, pages[at + p // h.page]) for p in range(key0, hi)]
            row_parts[r].append(part + r - row0 if part >= 0 else -1)
    used = set()
    for r in range(len(seen)):
        s, pos = flat[tokens[r // group, 2]]
        own = h.pages(s)
        assert sorted(seen[r]) == [(p, own[p // h.page]) for p in range(pos + 1)]
        if len(row_parts[r]) > 1:
            i = list(join_rows).index(r)
            assert sorted(join_parts[join_at[i]: join_at[i + 1]]) == sorted(row_parts[r])
            assert not used & set(row_parts[r])
            used |= set(row_parts[r])
        else:
            assert row_parts[r] == [-1] and r not in set(join_rows)
    assert len(used) == parts == next_part
    holders = {}
    for s in h.want:
        for p in h.pages(s):
            holders[int(p)] = holders.get(int(p), 0) + 1
    assert writable == all(holders[int(h.pages(s)[p // h.page])] == 1 for s, p in flat)
    return items, pages


@pytest.mark.parametrize("seed", range(16))
def test_plan_of_a_tree(lib, seed):
    r = random.Random(100 + seed)
    h = Host(lib, r.choice([16, 32, 64]), 4000, 40)
    root = h.new()
    h.extend([root], [r.randint(1, 900)])
    for _ in range(r.randint(1, 6)):
        _, kids = h.fork([r.choice(sorted(h.want)) for _ in range(r.randint(1, 4))], 0)
        h.extend(kids, [r.choice([0, 1, r.randint(0, 600)]) for _ in kids])
    lone = h.new()
    h.extend([lone], [r.randint(1, 2000)])
    seqs = sorted(h.want)
    r.shuffle(seqs)
    seqs = seqs[: r.randint(1, len(seqs))]
    n_new = [min(len(h.want[s]), r.choice([0, 1, 1, 2, r.randint(0, 60)])) for s in seqs]
    # (rows cheapest by the full tile, by 16 at a time, by 64)
    cost = r.choice([(47, 56, 59, 83), (65, 260, 262, 514), (46, 54, 60, 158), (10, 10, 10, 10)])
    check_plan(h, seqs, n_new, r.choice([1, 3, 4, 7, 40]), cost=cost, wgs=r.choice([8, 512, 4096]))


def test_a_shared_run_is_read_once(lib):
    h = Host(lib, 64, 1000, 70)
    root = h.new()
    h.extend([root], [64 * 100 + 20])
    _, kids = h.fork([root] * 64, 0)
    h.extend(kids, [1 + i for i in range(64)])
    items, pages = check_plan(h, kids, [1] * 64, 4, n_kv=8)
    assert len(pages) == 100 + sum(len(h.pages(s)) - 100 for s in kids)
    # a short run of few rows' worth is not worth its partial results; a chunk of many tokens neither
    h.extend(kids[:2], [500, 500])
    _, pages = check_plan(h, kids[:2], [500, 500], 4, n_kv=8)
    assert len(pages) == sum(len(h.pages(s)) for s in kids[:2])


@pytest.mark.parametrize("n,new", [(1, 1), (1, 0), (40, 40), (16, 1), (17, 16), (5000, 1), (5000, 700)])
def test_plan_of_one_sequence(lib, n, new):
    h = Host(lib, 16, 400, 2)
    a = h.new()
    h.extend([a], [n])
    if new == 0:
        tokens, items, *_ = plan(h, [a], [0], 4)
        assert len(tokens) == 0 and len(items) == 0
    else:
        check_plan(h, [a], [new], 4)


def test_pages_of_new_tokens_with_other_holders(lib):
    h = Host(lib, 32, 50, 4)
    a = h.new()
    h.extend([a], [40])
    h.fork([a], 0)
    *_, ((_, writable),) = plan(h, [a], [1], 1)
    assert not writable
    check_plan(h, [a], [9], 1)
