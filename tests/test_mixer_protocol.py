"""The barriers of the tensor-core linear attention kernel (csrc/linattn_tc.cu), role by role, on the CPU.

A role's steps and waits do not depend on what other roles do in between, so one run fixes the order that every run keeps
("happens before": a role's own order, and from a barrier phase's arrivals to its waits).  Over that order are checked, for
every number of chunks and both head sizes:

  * every role ends (in one run, hence in all);
  * a wait names its phase by parity alone, so the phase after it must need something that the waiting role does later; and
    an arrival must come after all of the phase before, or it would count for that one;
  * two accesses to the same columns of TMEM or tile of shared memory, one of them a write, are ordered.  A product starts
    somewhere behind its issue and has ended where a commit behind it is seen; two products execute in the order of their
    issue only where they add to the same accumulator.

The roles below restate those of la_tc_kernel line by line: who changes the one changes the other.
"""
import itertools

import pytest


class Model:
    def __init__(self, split, local, three, nc, DV, pv_done=True, order=None):
        self.split, self.local, self.three, self.nc = split, local, three, nc
        self.pv_done, self.order = pv_done, order
        self.NB, self.NW = DV // 64, DV // 32
        self.NA = 0 if local else 2 if split else 1
        self.NS = (6 if split else 3) if local else (4 if split else 2)
        self.DV = DV
        self.whole_x = split or local
        self.two_x = split and not local and not three
        # columns of TMEM, in blocks of 16
        self.inc_cols = 128 if split else DV
        self.c_x = 256 if local else 256 + self.inc_cols
        self.part = 32 if split else 64
        assert self.c_x + self.part * (3 if self.whole_x else 2) <= 512
        self.anc = []            # event -> bitmask of the events before it
        self.names = []
        self.access = []         # (first event, last event, region, write, kind, accumulator)
        self.waits = []          # (barrier, phase, event)
        self.bars = {}           # barrier -> arrivals of each phase, and the events in which phases complete
        self.products = []       # ends of the issuing warp's products

    # ---- events ----
    def event(self, name, *before):
        e = len(self.anc)
        m = 0
        for b in before:
            m |= self.anc[b] | (1 << b)
        self.anc.append(m)
        self.names.append(name)
        return e

    def before(self, a, b):
        return self.anc[b] >> a & 1

    def count(self, bar):
        b = bar[0]
        if b in ("OOUT", "P", "OS", "OFREE"):
            return 4
        if b in ("REL", "X", "X2", "ST"):
            return 4 * self.NW
        if b == "KV":    # the loading thread, and each tile's bytes
            return 1 + (3 if self.split and not self.local else 2)
        if b == "Q":
            return 2
        return 1

    def arrive(self, bar, event):
        st = self.bars.setdefault(bar, dict(arrivals=[[]], done=[]))
        if len(st["arrivals"][-1]) == self.count(bar):
            st["arrivals"].append([])
        st["arrivals"][-1].append(event)
        if len(st["arrivals"][-1]) == self.count(bar):
            st["done"].append(self.event(f"{bar} phase {len(st['done'])}", *st["arrivals"][-1]))

    # ---- regions ----
    def cols(self, first, n, quads=range(4)):
        return [("tmem", c, q) for c in range(first // 16, (first + n + 15) // 16) for q in quads]

    def tile(self, what, stage, parts):
        return [(what, stage, p) for p in parts]

    def c_p(self, a):
        return a * 128

    def c_o(self, a):
        return a * 128 + 64 if self.split else 128

    def c_inc(self, c):
        return (c & 1) * 128 if self.local else 256

    def x_col(self, c):
        return self.c_x + ((c & 1) * 64 if self.two_x else 0)

    def x_bar(self, c):
        return ("X2",) if self.split and not self.local and c & 1 else ("X",)

    def x_ph(self, c):
        return c >> 1 if self.split and not self.local else c

    def grp(self, c):
        return c % self.NA if self.NA else 0

    # ---- roles: generators of ("wait", barrier, phase) and of calls with the role's last event ----
    def loader(self):
        nc, NS, split = self.nc, self.NS, self.split
        kv = qs = 0
        stores = []

        def load(what, c, bar):
            def do(last):
                e = self.event(f"load {what}{c}", last)
                d = self.event(f"{what}{c} there", e)
                self.access += [(e, d, r, True, "load", None) for r in self.tile(what, c % NS, range(16))]
                self.arrive(bar, d)
                return e
            return ("do", do)

        def expect(bar):
            return ("arrive", bar)

        def load_kv(c):
            yield expect(("KV", c % NS))
            yield load("K", c, ("KV", c % NS))
            yield load("V", c, ("KV", c % NS))

        def load_q(c):
            bar = ("KV" if split else "Q", c % NS)
            if not split:
                yield expect(bar)
            yield load("Q", c, bar)

        def store(c):
            def do(last):
                e = self.event(f"store O{c}", last)
                d = self.event(f"O{c} read", e)
                stores.append(d)
                self.access += [(e, d, r, False, "store", None) for r in self.tile("Q", c % NS, range(16))]
                return e
            return ("do", do)

        def stores_read():
            return ("do", lambda last: self.event("stores read", last, *stores))

        while kv < min(nc, NS):
            yield from load_kv(kv)
            kv += 1
            if not self.local:
                yield from load_q(qs)
                qs += 1
        for c in range(nc):
            r = c % NS
            if self.local:
                yield ("wait", ("PV", r), c // NS)
                if kv < nc:
                    yield from load_kv(kv)
                    kv += 1
                continue
            if not split:
                yield ("wait", ("REL", r), c // NS)
                yield ("wait", ("PV", r), c // NS)
                if kv < nc:
                    yield from load_kv(kv)
                    kv += 1
            yield ("wait", ("OOUT", r), c // NS)
            yield store(c)
            if qs < nc:
                if split:
                    yield ("wait", ("REL", r), c // NS)
                yield stores_read()
                if split:
                    yield from load_kv(kv)
                    kv += 1
                yield from load_q(qs)
                qs += 1

    def issuer(self):
        nc, NS, NA, split, local = self.nc, self.NS, self.NA, self.split, self.local
        later = self.three and not self.whole_x

        def product(name, acc, reads, writes):
            def do(last):
                e = self.event("issue " + name, last)
                d = self.event(name + " done", e)
                self.products.append(d)
                self.access += [(e, d, r, False, "mma", acc) for r in reads]
                self.access += [(e, d, r, True, "mma", acc) for r in writes]
                return e
            return ("do", do)

        def commit(*bar):
            return ("do", lambda last: (self.arrive(bar, self.event(f"commit {bar}", last, *self.products)), last)[1])

        def q_k_waits(c):
            yield ("wait", ("KV", c % NS), c // NS)
            if not split:
                yield ("wait", ("Q", c % NS), c // NS)
                if c > 0 and self.pv_done:
                    yield ("wait", ("O", 0), c - 1)
            if split and c >= NA:
                yield ("wait", ("OFREE", self.grp(c)), (c - NA) // NA)

        def q_k_issue(c):
            p = self.c_p(self.grp(c))
            yield product(f"QK{c}", ("P", self.grp(c)), self.tile("Q", c % NS, range(16)) + self.tile("K", c % NS, range(16)),
                          self.cols(p, 128))
            yield commit("S", self.grp(c))

        def q_k(c):
            yield from q_k_waits(c)
            yield from q_k_issue(c)

        def q_s_waits(c):
            if split:
                yield ("wait", ("P", self.grp(c)), c // NA)
            elif c > 0:
                yield ("wait", ("OFREE", 0), c - 1)

        def q_s_issue(c):
            yield product(f"QS{c}", ("O", self.grp(c)), self.tile("Q", c % NS, range(16)) + self.tile("S", 0, range(16)),
                          self.cols(self.c_o(self.grp(c)), self.DV))
            yield commit("O1", self.grp(c))

        def q_s(c):
            yield from q_s_waits(c)
            yield from q_s_issue(c)

        def p_v(c):
            a = self.grp(c)
            yield ("wait", ("OS", a), c // NA)
            yield product(f"PV{c}", ("O", a), self.cols(self.c_p(a), 64) + self.tile("V", c % NS, range(16)),
                          self.cols(self.c_o(a), self.DV))
            yield commit("O", a)
            if not split:
                yield commit("PV", c % NS)

        def increment(c, at, parts):
            return product(f"XV{c}", ("INC", self.c_inc(c)), self.cols(at, parts * self.part) + self.tile("V", c % NS, range(16)),
                           self.cols(self.c_inc(c), self.inc_cols))

        def x_v(c):
            if local:
                yield ("wait", ("KV", c % NS), c // NS)
            yield ("wait", self.x_bar(c), self.x_ph(c))
            if not local:
                yield ("wait", ("ST",), c)
            yield increment(c, self.x_col(c), 3 if self.whole_x and self.three else 2)
            yield commit("INC")
            if local:
                yield commit("PV", c % NS)

        def x_v_third(c):
            yield ("wait", ("X2",), c)
            yield increment(c, self.c_x, 1)
            yield commit("INC2")

        if local:
            for c in range(nc):
                yield from x_v(c)
        elif split:
            if nc:
                yield from q_k(0)
            for c in range(nc):
                yield from x_v(c)
                if self.order == "one block" and c + 1 < nc:   # Q S and the next Q K^T issued together
                    yield from q_s_waits(c)
                    yield from q_k_waits(c + 1)
                    yield from q_s_issue(c)
                    yield from q_k_issue(c + 1)
                else:
                    yield from q_s(c)
                    if c + 1 < nc:
                        yield from q_k(c + 1)
                yield from p_v(c)
        else:
            for c in range(nc):
                yield from q_k(c)
                yield from x_v(c)
                yield from q_s(c)
                yield from p_v(c)
                if later:
                    yield from x_v_third(c)

    def output_warp(self, a, quad):
        NA, NS = self.NA, self.NS

        def touch(name, reads, writes):
            def do(last):
                e = self.event(name, last)
                self.access += [(e, e, r, False, "warp", None) for r in reads] + [(e, e, r, True, "warp", None) for r in writes]
                return e
            return ("do", do)

        for c in range(a, self.nc, NA):
            ph = c // NA
            yield ("wait", ("S", a), ph)
            yield touch(f"P{c}.{quad}", self.cols(self.c_p(a), 128, [quad]), self.cols(self.c_p(a), 64, [quad]))
            yield ("arrive", ("P", a))
            yield ("wait", ("O1", a), ph)
            yield touch(f"scale{c}.{quad}", [], self.cols(self.c_o(a), self.DV, [quad]))
            yield ("arrive", ("OS", a))
            yield ("wait", ("O", a), ph)
            yield touch(f"O{c}.{quad}", self.cols(self.c_o(a), self.DV, [quad]), self.tile("Q", c % NS, [quad]))
            yield ("arrive", ("OFREE", a))
            yield ("arrive", ("OOUT", c % NS))

    def state_warp(self, wg, quad):
        nc, NS, NW, split, local = self.nc, self.NS, self.NW, self.split, self.local

        def touch(name, reads, writes):
            def do(last):
                e = self.event(name, last)
                self.access += [(e, e, r, False, "warp", None) for r in reads] + [(e, e, r, True, "warp", None) for r in writes]
                return e
            return ("do", do)

        mine = (64 if split else 128) // NW     # positions whose X the warp makes
        xcol = wg * mine // 2

        def make_x(c, parts):
            w = [r for p in parts for r in self.cols(self.x_col(c) + (0 if parts == [2] else p) * self.part + xcol, mine // 2, [quad])]
            return touch(f"X{c}.{wg}.{quad}", self.tile("K", c % NS, range(16)), w)

        def give_x(c):
            yield ("wait", ("KV", c % NS), c // NS)
            yield touch(f"V{c} cut {wg}", [], self.tile("V", c % NS, [4 * wg + quad]))
            yield make_x(c, [0, 1, 2] if self.whole_x and self.three else [0, 1])
            yield ("arrive", self.x_bar(c))

        def publish(c):
            return touch(f"S{c}.{wg}.{quad}", [], self.tile("S", 0, [4 * wg + quad]))

        def take(c):
            first = self.c_inc(c) + ((quad >> 1) * 64 if split else 0) + wg * 32
            return touch(f"take{c}.{wg}.{quad}", self.cols(first, 32, [quad]), [])

        if not local:
            yield publish(-1)
            yield ("arrive", ("ST",))
        if nc > 0:
            yield from give_x(0)
        for c in range(nc):
            if self.two_x and c + 1 < nc:
                yield from give_x(c + 1)
            yield ("wait", ("INC",), c)
            if self.three and not self.whole_x:
                yield make_x(c, [2])
                yield ("arrive", ("X2",))
                yield ("wait", ("INC2",), c)
            if not self.two_x and c + 1 < nc:
                yield from give_x(c + 1)
            if not local:
                yield ("wait", ("O1", self.grp(c)), c // self.NA)
            yield take(c)
            if local:
                continue
            if c + 1 < nc:
                yield publish(c)
            yield ("arrive", ("ST",))
            yield ("arrive", ("REL", c % NS))

    # ---- a run, and its checks ----
    def run(self):
        roles = {"loader": self.loader(), "issuer": self.issuer()}
        roles.update({f"output {a}.{q}": self.output_warp(a, q) for a in range(self.NA) for q in range(4)})
        roles.update({f"state {w}.{q}": self.state_warp(w, q) for w in range(self.NW) for q in range(4)})
        begin = self.event("begin")
        last = {r: begin for r in roles}
        ahead = {r: next(g, None) for r, g in roles.items()}
        while any(s is not None for s in ahead.values()):
            moved = False
            for r, g in roles.items():
                while ahead[r] is not None:
                    s = ahead[r]
                    if s[0] == "wait":
                        done = self.bars.get(s[1], dict(done=[]))["done"]
                        if len(done) <= s[2]:
                            break
                        last[r] = self.event(f"{r} waits {s[1]} {s[2]}", last[r], done[s[2]])
                        self.waits.append((s[1], s[2], last[r]))
                    elif s[0] == "arrive":
                        last[r] = self.event(f"{r} arrives {s[1]}", last[r])
                        self.arrive(s[1], last[r])
                    else:
                        last[r] = s[1](last[r])
                    ahead[r] = next(g, None)
                    moved = True
            if not moved:
                return [f"stuck: {r} at {s[1]} phase {s[2]}" for r, s in ahead.items() if s is not None]
        return self.faults()

    def faults(self):
        out = []
        for bar, phase, w in self.waits:
            done = self.bars[bar]["done"]
            if len(done) > phase + 1 and not self.before(w, done[phase + 1]):
                out.append(f"{self.names[w]}: the next phase may complete first")
        for bar, st in self.bars.items():
            for p, arrivals in enumerate(st["arrivals"][1:]):
                for e in arrivals:
                    if not all(self.before(a, e) for a in st["arrivals"][p]):
                        out.append(f"{self.names[e]} may count for phase {p}")
        at = {}
        for a in self.access:
            at.setdefault(a[2], []).append(a)
        for region, acc in at.items():
            for a, b in itertools.combinations(acc, 2):
                if not (a[3] or b[3]) or a[:2] == b[:2]:
                    continue
                if a[4] == b[4] == "mma" and a[5] == b[5]:   # in the order of their issue
                    continue
                if not (a[1] == b[0] or b[1] == a[0] or self.before(a[1], b[0]) or self.before(b[1], a[0])):
                    out.append(f"{region}: {self.names[a[0]]} and {self.names[b[0]]}")
        return out


SHAPES = [dict(split=True, local=False, three=False, DV=64), dict(split=True, local=False, three=True, DV=64),
          dict(split=False, local=False, three=False, DV=128), dict(split=False, local=False, three=True, DV=128),
          dict(split=False, local=False, three=False, DV=64), dict(split=False, local=False, three=True, DV=64),
          dict(split=True, local=True, three=True, DV=64), dict(split=False, local=True, three=True, DV=128),
          dict(split=False, local=True, three=True, DV=64)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(f"{k}{int(v)}" for k, v in s.items()))
@pytest.mark.parametrize("nc", [0, 1, 2, 3, 4, 5, 8, 13])
def test_roles_end_and_their_accesses_are_ordered(shape, nc):
    assert Model(nc=nc, **shape).run() == []


def test_a_missing_wait_is_seen():
    """Q K^T of a chunk goes where P of the chunk before lies, which P V reads: without a wait for that product nothing
    orders the two, whose accumulators differ."""
    faults = Model(nc=3, pv_done=False, **SHAPES[2]).run()
    assert faults and all("PV" in f and "QK" in f for f in faults)


@pytest.mark.parametrize("shape", SHAPES[:2], ids=["two parts", "three parts"])
def test_the_order_is_free_of_faults_with_two_products_issued_together(shape):
    """Q S and the next chunk's Q K^T issued behind all their waits at once, as an earlier form of the kernel had it."""
    for nc in (2, 5, 13):
        assert Model(nc=nc, order="one block", **shape).run() == []
