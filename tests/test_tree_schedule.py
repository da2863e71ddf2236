"""CPU model of the tree attention kernel's roles and barriers.

Each role of csrc/sas_tree.cu is a generator that yields the barrier and parity
it waits for and arrives where the kernel does; copies and MMAs complete later,
MMAs in the order they were issued, everything else in a random order. A
barrier's parity wait passes when the phase of that parity is the last one
completed, as the hardware's does, so a waiter that is overtaken by two phases
blocks. The model checks that no tile sequence blocks, and that no buffer is
written while a reader is still to come: each buffer holds the tile that its
readers expect.
"""

import random

import pytest

RING, UNIT_SLOTS = 4, 6
FIRST, LAST, END, ZERO = 1, 2, 4, 8


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def done(self, parity):
        return (self.phase & 1) != (parity & 1)


class Cta:
    """One side of the pair; a warp group (8 loader warps, 4 softmax warps) is one role."""

    def __init__(self):
        names = dict(kfull=1, vfull=1, qfull=1, xk=1, xv=1, xq=1, kempty=1, vempty=1, qempty=1, pready=2, ofull=1, oempty=2)
        self.b = {k: Bar(v) for k, v in names.items()}
        for i in range(3):
            self.b[f"mask{i}"] = Bar(1)
        for i in range(2):
            self.b[f"sfull{i}"] = Bar(1)
        for i in range(RING):
            self.b[f"cfull{i}"], self.b[f"cempty{i}"] = Bar(1), Bar(3)  # loaders, MMA, softmax
        self.ring, self.units = [None] * RING, [None] * UNIT_SLOTS
        self.mask, self.s = [None] * 3, [None] * 2
        self.k = self.v = self.q = self.p = self.o = None


class Model:
    def __init__(self, units, seed):
        """units: a list of tile counts, 0 for a unit without a used token."""
        self.rng, self.units = random.Random(seed), units
        self.cta = [Cta(), Cta()]
        self.mmas, self.copies = [], []  # pending completions; MMAs in order
        self.tiles_done = [0, 0]

    def commit(self, *bars):
        self.mmas.append(lambda: [c.b[x].arrive() for c in self.cta for x in bars])

    def coordinator(self, side):
        c, n, b = 0, 0, self.cta[side].b
        seq = self.units + [None]
        uc = 0
        for u, tiles in enumerate(seq):
            entries = [(END, None)] if tiles is None else [(ZERO, None)] if tiles == 0 else \
                [((FIRST if k == 0 else 0) | (LAST if k == tiles - 1 else 0), k) for k in range(tiles)]
            yield f"cempty{c % RING}", c // RING + 1
            self.cta[side].units[uc % UNIT_SLOTS] = u
            for fl, _ in entries:
                yield f"cempty{c % RING}", c // RING + 1
                tile = None if fl & (END | ZERO) else n
                n += tile is not None
                self.cta[side].ring[c % RING] = (fl, tile, u, uc % UNIT_SLOTS)
                b[f"cfull{c % RING}"].arrive()
                c += 1
            uc += 1

    def loader(self, side):
        me, b = self.cta[side], self.cta[side].b
        c = n = q = 0
        due = None

        def load_v(m, u):
            yield "vempty", m + 1
            self.copies.append(lambda: (setattr(me, "v", (m, u)), b["vfull"].arrive()))

        while True:
            yield f"cfull{c % RING}", c // RING
            fl, tile, u, us = me.ring[c % RING]
            if fl & (END | ZERO):
                if due:
                    yield from load_v(*due)
                due = None
                if fl & END:
                    return
            else:
                assert tile == n and me.units[us] == u
                if fl & FIRST:
                    yield "qempty", q + 1
                    self.copies.append(lambda u=u: (setattr(me, "q", u), b["qfull"].arrive()))
                    q += 1
                yield "kempty", n + 1
                me.mask[n % 3] = n
                b[f"mask{n % 3}"].arrive()
                self.copies.append(lambda n=n, u=u: (setattr(me, "k", (n, u)), b["kfull"].arrive()))
                if due:
                    yield from load_v(*due)
                due = (n, u)
                n += 1
            b[f"cempty{c % RING}"].arrive()
            c += 1

    def mma(self, side):
        me, first = self.cta[side], self.cta[0]
        c = n = u_count = vu = 0
        due = None

        def pass_on(bar, to, par):
            yield bar, par
            first.b[to].arrive()

        def product(m, fl, u):
            nonlocal vu
            if side:
                yield from pass_on("vfull", "xv", m)
                return
            yield "pready", m
            yield "vfull", m
            yield "xv", m
            if fl & FIRST:
                yield "oempty", vu + 1

            def run():
                for cta in self.cta:
                    assert cta.v == (m, u) and cta.p == m
                    assert (cta.o is None) if fl & FIRST else cta.o[0] == u and cta.o[1] == m - 1
                    cta.o = (u, m)
            self.mmas.append(run)
            self.commit("vempty")
            if fl & LAST:
                self.commit("ofull")
                vu += 1

        while True:
            yield f"cfull{c % RING}", c // RING
            fl, tile, u, _ = me.ring[c % RING]
            if fl & (END | ZERO):
                if due:
                    yield from product(*due)
                due = None
                if fl & END:
                    return
            else:
                if side:
                    if fl & FIRST:
                        yield from pass_on("qfull", "xq", u_count)
                        u_count += 1
                    yield from pass_on("kfull", "xk", n)
                else:
                    if fl & FIRST:
                        yield "qfull", u_count
                        yield "xq", u_count
                        u_count += 1
                    yield "kfull", n
                    yield "xk", n

                    def run(n=n, u=u):
                        for cta in self.cta:
                            assert cta.k == (n, u) and cta.q == u
                            assert cta.s[n & 1] is None, "scores overwritten before they were read"
                            cta.s[n & 1] = n
                    self.mmas.append(run)
                    self.commit(f"sfull{n & 1}", "kempty")
                    if fl & LAST:
                        self.commit("qempty")
                if due:
                    yield from product(*due)
                due = (n, fl, u)
                n += 1
            me.b[f"cempty{c % RING}"].arrive()
            c += 1

    def softmax(self, side):
        me, first = self.cta[side], self.cta[0]
        c = n = done = 0
        while True:
            yield f"cfull{c % RING}", c // RING
            fl, tile, u, us = me.ring[c % RING]
            if fl & END:
                return
            assert me.units[us] == u, "a unit's slot was rewritten"
            if not fl & ZERO:
                yield f"mask{n % 3}", n // 3
                yield f"sfull{n & 1}", n >> 1
                assert me.mask[n % 3] == n and me.s[n & 1] == n
                me.s[n & 1] = None
                if self.rng.random() < 0.2:  # rows that are not finite: V has to be there
                    yield "vempty", n + 1
                    yield "vfull", n
                    assert me.v == (n, u)
                yield "vempty", n + 1
                me.p = n
                first.b["pready"].arrive()
                n += 1
                if fl & LAST:
                    yield "ofull", done
                    done += 1
                    assert me.o == (u, n - 1)
                    me.o = None
                    first.b["oempty"].arrive()
            me.b[f"cempty{c % RING}"].arrive()
            c += 1

    def run(self):
        roles = [(s, f(s)) for s in (0, 1) for f in (self.coordinator, self.loader, self.mma, self.softmax)]
        waits = {i: next(g, None) for i, (s, g) in enumerate(roles)}
        live = {i for i, w in waits.items() if w}
        while live:
            ready = [i for i in live if self.cta[roles[i][0]].b[waits[i][0]].done(waits[i][1])]
            events = ready + (["mma"] if self.mmas else []) + (["copy"] if self.copies else [])
            assert events, f"blocked: {[(roles[i][0], roles[i][1].__name__, waits[i]) for i in live]}"
            e = self.rng.choice(events)
            if e == "mma":
                self.mmas.pop(0)()
            elif e == "copy":
                self.copies.pop(self.rng.randrange(len(self.copies)))()
            else:
                try:
                    waits[e] = next(roles[e][1])
                except StopIteration:
                    live.discard(e)
        while self.mmas:
            self.mmas.pop(0)()


@pytest.mark.parametrize("seed", range(60))
def test_no_sequence_blocks(seed):
    r = random.Random(seed)
    units = [r.choice([0, 0, 1, 1, 2, 3, 7]) for _ in range(r.randrange(0, 14))]
    Model(units, seed).run()


@pytest.mark.parametrize("units", [[], [0] * 9, [1] + [0] * 9 + [1], [2] + [0] * 5, [0] * 6 + [1], [1] * 12, [13]])
def test_edges(units):
    for seed in range(10):
        Model(units, seed).run()
