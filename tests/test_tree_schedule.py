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

RING, UNIT_SLOTS = 7, 9
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
    """One side of the pair; a group of warps with one task is one role."""

    def __init__(self):
        names = dict(qfull=1, xq=1, qempty=1, pready=2, ofull=1)
        names.update({f"{k}{h}": 1 for k in ("kfull", "vfull", "xk", "xv", "kempty", "vempty") for h in (0, 1)})  # halves of K, V
        names.update({f"{k}{i}": c for k, n, c in (("mask", 3, 1), ("sfull", 2, 1), ("sempty", 2, 2), ("oempty", 3, 2), ("fin", 2, 1), ("cfull", RING, 1),
                                                   ("cempty", RING, 5)) for i in range(n)})  # K, V, scores, products, softmax
        self.b = {k: Bar(v) for k, v in names.items()}
        self.ring, self.units = [None] * RING, [None] * UNIT_SLOTS
        self.mask, self.s, self.fin = [None] * 3, [None] * 2, [None] * 2
        self.k, self.v = [None] * 2, [None] * 2
        self.q = self.p = None
        self.o = [None] * 3  # places of halves of O, in turn
        self.out = []


class Model:
    def __init__(self, units, seed):
        """units: a list of tile counts, 0 for a unit without a used token."""
        self.rng, self.units = random.Random(seed), units
        self.cta = [Cta(), Cta()]
        self.mmas, self.copies = {"qk": [], "pv": []}, []  # pending completions; each issuer's MMAs in order

    def commit(self, q, *bars):
        self.mmas[q].append(lambda: [c.b[x].arrive() for c in self.cta for x in bars])

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

    def walk(self, side, on_tile, on_end=None):
        """The ring as every role walks it; on_tile(tile, unit, flags, slot) for tiles with rows."""
        me, c = self.cta[side], 0
        while True:
            yield f"cfull{c % RING}", c // RING
            fl, tile, u, us = me.ring[c % RING]
            if fl & END:
                if on_end:
                    yield from on_end()
                return
            if not fl & ZERO:
                assert me.units[us] == u, "a unit's slot was rewritten"
                yield from on_tile(tile, u, fl)
                assert me.units[us] == u, "a unit's slot was rewritten"
            me.b[f"cempty{c % RING}"].arrive()
            c += 1

    def k_loader(self, side):
        me, b, q = self.cta[side], self.cta[side].b, [0]

        def tile(n, u, fl):
            if fl & FIRST:
                yield "qempty", q[0] + 1
                self.copies.append(lambda: (setattr(me, "q", u), b["qfull"].arrive()))
                q[0] += 1
            for h in (0, 1):
                yield f"kempty{h}", n + 1
                self.copies.append(lambda h=h: (me.k.__setitem__(h, (n, u)), b[f"kfull{h}"].arrive()))
                if h == 0:
                    assert me.mask[n % 3] is None, "a mask was overwritten before it was read"
                    me.mask[n % 3] = n
                    b[f"mask{n % 3}"].arrive()
        yield from self.walk(side, tile)

    def v_loader(self, side):
        me, b = self.cta[side], self.cta[side].b

        def tile(n, u, fl):
            for h in (0, 1):
                yield f"vempty{h}", n + 1
                self.copies.append(lambda h=h: (me.v.__setitem__(h, (n, u)), b[f"vfull{h}"].arrive()))
        yield from self.walk(side, tile)

    def pass_on(self, bar, to, par):
        yield bar, par
        self.cta[0].b[to].arrive()

    def scores(self, side):
        units = [0]

        def tile(n, u, fl):
            if side:
                if fl & FIRST:
                    yield from self.pass_on("qfull", "xq", units[0])
                    units[0] += 1
                for h in (0, 1):
                    yield from self.pass_on(f"kfull{h}", f"xk{h}", n)
                return
            if fl & FIRST:
                yield "qfull", units[0]
                yield "xq", units[0]
                units[0] += 1
            yield f"sempty{n & 1}", (n >> 1) + 1
            for h in (0, 1):
                yield f"kfull{h}", n
                yield f"xk{h}", n

                def run(h=h):
                    for cta in self.cta:
                        assert cta.k[h] == (n, u) and cta.q == u
                        assert cta.s[n & 1] == (n if h else None), "scores overwritten before they were read"
                        cta.s[n & 1] = n
                self.mmas["qk"].append(run)
                self.commit("qk", f"kempty{h}")
            self.commit("qk", f"sfull{n & 1}")
            if fl & LAST:
                self.commit("qk", "qempty")
        yield from self.walk(side, tile)

    def products(self, side):
        done = [0]

        def tile(n, u, fl):
            if side:
                for h in (0, 1):
                    yield from self.pass_on(f"vfull{h}", f"xv{h}", n)
                return
            yield "pready", n
            for h in (0, 1):
                use, place = divmod(2 * done[0] + h, 3)
                if fl & FIRST:
                    yield f"oempty{place}", use + 1
                yield f"vfull{h}", n
                yield f"xv{h}", n

                def run(h=h, place=place):
                    for cta in self.cta:
                        assert cta.v[h] == (n, u) and cta.p == n
                        assert cta.o[place] == (None if fl & FIRST else (u, n - 1, h)), "O overwritten before it was read"
                        cta.o[place] = (u, n, h)
                self.mmas["pv"].append(run)
                self.commit("pv", f"vempty{h}")
            if fl & LAST:
                self.commit("pv", "ofull")
                done[0] += 1
        yield from self.walk(side, tile)

    def softmax(self, side):
        me, first, st = self.cta[side], self.cta[0], dict(n=0, u=0)

        def tile(n, u, fl):
            assert n == st["n"]
            yield f"mask{n % 3}", n // 3
            assert me.mask[n % 3] == n
            me.mask[n % 3] = None
            yield f"sfull{n & 1}", n >> 1
            assert me.s[n & 1] == n
            me.s[n & 1] = None
            first.b[f"sempty{n & 1}"].arrive()
            if self.rng.random() < 0.2:  # rows that are not finite: V has to be there
                yield "vempty1", n + 1
                for h in (0, 1):
                    yield f"vfull{h}", n
                assert me.v == [(n, u)] * 2
            yield "vempty1", n + 1
            me.p = n
            first.b["pready"].arrive()
            st["n"] += 1
            if fl & LAST:
                self.finish(me, st["u"], (u, n))
                st["u"] += 1

        def end():
            if st["n"]:
                yield "vempty1", st["n"] + 1
            self.finish(me, st["u"], END)
        yield from self.walk(side, tile, end)

    def finish(self, me, u, what):
        assert me.fin[u & 1] is None, "a finished unit's place was rewritten"
        me.fin[u & 1] = what
        me.b[f"fin{u & 1}"].arrive()

    def epilogue(self, side):
        me, u = self.cta[side], 0
        while True:
            yield f"fin{u & 1}", u >> 1
            what, me.fin[u & 1] = me.fin[u & 1], None
            if what == END:
                return
            yield "ofull", u
            for h in (0, 1):
                place = (2 * u + h) % 3
                assert me.o[place] == (*what, h)
                me.o[place] = None
                self.cta[0].b[f"oempty{place}"].arrive()
                yield None, 0  # others may run in between
            me.out.append(what[0])
            u += 1

    def run(self):
        kinds = (self.coordinator, self.k_loader, self.v_loader, self.scores, self.products, self.softmax, self.epilogue)
        roles = [(s, f(s)) for s in (0, 1) for f in kinds]
        waits = {i: next(g, None) for i, (s, g) in enumerate(roles)}
        live = {i for i, w in waits.items() if w}
        bias = self.rng.choice([None, *range(len(roles))])  # one role is slow, or none
        while live:
            ready = [i for i in live if waits[i][0] is None or self.cta[roles[i][0]].b[waits[i][0]].done(waits[i][1])]
            events = ready + [q for q in self.mmas if self.mmas[q]] + (["copy"] if self.copies else [])
            assert events, f"blocked: {[(roles[i][0], kinds[i % len(kinds)].__name__, waits[i]) for i in live]}"
            e = self.rng.choice([x for x in events if x != bias] or events)
            if e in self.mmas:
                self.mmas[e].pop(0)()
            elif e == "copy":
                self.copies.pop(self.rng.randrange(len(self.copies)))()
            else:
                try:
                    waits[e] = next(roles[e][1])
                except StopIteration:
                    live.discard(e)
        for cta in self.cta:
            assert cta.out == [u for u, tiles in enumerate(self.units) if tiles]


@pytest.mark.parametrize("seed", range(120))
def test_no_sequence_blocks(seed):
    r = random.Random(seed)
    units = [r.choice([0, 0, 1, 1, 2, 3, 7]) for _ in range(r.randrange(0, 14))]
    Model(units, seed).run()


@pytest.mark.parametrize("units", [[], [0] * 9, [1] + [0] * 9 + [1], [2] + [0] * 5, [0] * 6 + [1], [1] * 12, [13]])
def test_edges(units):
    for seed in range(25):
        Model(units, seed).run()


class TxBar(Bar):
    """A barrier whose phase also waits for the bytes (here: boxes) that it was told to expect."""

    def __init__(self, count):
        super().__init__(count)
        self.tx = 0

    def arrive(self, n=1):
        self.left -= n
        assert self.left >= 0, "an arrival too many"
        self.check()

    def expect(self):
        self.tx += 1

    def landed(self):
        self.tx -= 1
        self.check()

    def check(self):
        if self.left == 0 and self.tx == 0:
            self.left, self.phase = self.count, self.phase + 1


class Loaders:
    """The four warps that copy K (or V) in halves, a reader, and a wait that gives up at some moment. Afterwards every
    wait may give up, or pass if its phase is complete. By boxes, warp 0 alone copies; else each warp its rows, which
    arrive by themselves once they have landed. ``rule`` is how a warp leaves."""

    def __init__(self, tiles, seed, rule):
        self.rng, self.tiles, self.rule = random.Random(seed), tiles, rule
        self.full, self.empty = [TxBar(4), TxBar(4)], [Bar(1), Bar(1)]
        self.flying, self.abort, self.sent, self.left = [], False, None, 0
        self.blocked = False

    def wait(self, bar, parity):
        while True:
            if bar.done(parity) and (not self.abort or self.rng.random() < 0.5):
                return True
            if self.abort and self.rng.random() < 0.5:
                return bar.done(parity)
            yield

    def loader(self, w):
        done = [0, 0]
        for n, boxes in enumerate(self.tiles):
            for h in (0, 1):
                if not (yield from self.wait(self.empty[h], n + 1)):
                    yield from self.leave(w, done)
                    return
                if boxes:
                    if w == 0:
                        self.full[h].expect()
                        self.flying.append((w, self.full[h].landed))
                    yield
                    self.full[h].arrive()
                else:
                    self.flying.append((w, self.full[h].arrive))
                done[h] += 1
                yield
        yield from self.leave(w, done)

    def leave(self, w, done):
        while any(x == w and land.__name__ == "arrive" for x, land in self.flying):  # cp.async.wait_all
            yield
        if self.rule == "whole tiles":
            if w == 0 and done[1]:
                for h in (0, 1):
                    yield from self.drain(self.full[h], done[1] - 1)
        else:
            if w == 0:
                self.sent = list(done)
            self.left += 1
            while self.left < 4:
                yield
            for h in (0, 1):
                if done[h] < self.sent[h]:
                    assert done[h] == self.sent[h] - 1
                    self.full[h].arrive()
                if w == 0 and self.sent[h]:
                    yield from self.drain(self.full[h], self.sent[h] - 1)
        if w == 0:
            assert not self.flying, "a copy is still landing"

    def drain(self, bar, parity):
        while not bar.done(parity):
            self.blocked = not self.flying and self.left == 4
            assert not self.blocked or self.idle < 200, "the drain waits for a phase that cannot end"
            yield

    def reader(self):
        for n in range(len(self.tiles)):
            for h in (0, 1):
                if not (yield from self.wait(self.full[h], n)):
                    return
                yield
                self.empty[h].arrive()

    def run(self):
        roles = [self.loader(w) for w in range(4)] + [self.reader()]
        at, step, self.idle = self.rng.randrange(1, 60), 0, 0
        while roles or self.flying:
            step += 1
            self.abort = self.abort or step >= at
            self.idle = 0 if self.flying else self.idle + 1
            if self.flying and (not roles or self.rng.random() < 0.1):
                self.flying.pop(self.rng.randrange(len(self.flying)))[1]()
            else:
                g = self.rng.choice(roles)
                try:
                    next(g)
                except StopIteration:
                    roles.remove(g)
            assert step < 100000, "blocked"


def _loaders(seed, rule):
    r = random.Random(seed)
    boxes = r.choice([True, True, None])
    Loaders([r.random() < 0.5 if boxes is None else boxes for _ in range(r.randrange(1, 12))], seed, rule).run()


@pytest.mark.parametrize("block", range(8))
def test_no_copy_lands_after_a_wait_gave_up(block):
    for seed in range(250 * block, 250 * block + 250):
        _loaders(seed, "halves sent")


def test_counting_whole_tiles_leaves_copies_in_flight():
    """The model tells: a warp that waits for its last whole tile leaves while a first half is landing."""
    found = 0
    for seed in range(400):
        try:
            _loaders(seed, "whole tiles")
        except AssertionError as e:
            found += "still landing" in str(e)
    assert found > 0


class LateCommits(Model):
    """Commits that reach the second CTA's barriers later than the first's, each issuer's in order. ``both``: the second
    CTA's issuers wait for the first's last one, as the kernel's do."""

    def __init__(self, units, seed, both):
        super().__init__(units, seed)
        self.both, self.late = both, {"qk": [], "pv": []}
        for cta in self.cta:
            cta.b.update(drainqk=Bar(1), drainpv=Bar(1))

    def commit(self, q, *bars):
        def done():
            for x in bars:
                self.cta[0].b[x].arrive()
                self.late[q].append(self.cta[1].b[x].arrive)
                self.copies.append(lambda: self.late[q].pop(0)())
        self.mmas[q].append(done)

    def issuer(self, q, side, role):
        yield from role(side)
        if side == 0:
            self.commit(q, f"drain{q}")
        if side == 0 or self.both:
            yield f"drain{q}", 0

    def scores(self, side):
        return self.issuer("qk", side, super().scores)

    def products(self, side):
        return self.issuer("pv", side, super().products)


@pytest.mark.parametrize("both", [True, False])
def test_no_commit_arrives_after_the_pair_left(both):
    found = 0
    for seed in range(300):
        r = random.Random(seed)
        m = LateCommits([r.choice([0, 1, 1, 2, 3]) for _ in range(r.randrange(1, 6))], seed, both)
        m.run()
        found += bool(m.late["qk"] or m.late["pv"])
    assert found == 0 if both else found > 0


def test_the_model_has_the_kernels_constants():
    import os
    import re

    with open(os.path.join(os.path.dirname(__file__), "..", "dsv4_b200", "csrc", "sas_tree.cu")) as f:
        source = f.read()
    const = lambda name: int(re.search(rf"constexpr int (?:[^;]*,\s+)?{name} = (\d+)", source).group(1))  # noqa: E731
    assert (const("kRing"), const("kUnitSlots"), const("kLoadWarps")) == (RING, UNIT_SLOTS, 4)
