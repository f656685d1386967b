"""The prompt kernel's barriers (csrc/prompt.cu) as a small model on the CPU.

An mbarrier wait knows the parity of a phase only, so a wait for phase f also
passes while the barrier still is one phase short of it.  The model keeps
parities as the hardware does, lands TMA loads in any order, runs the tensor
pipe late, and lets every role go on at random.  It checks that each product and
each row warp's look at a V tile meets the tile that it means, that no stage is
loaded over a tile in use, and that nothing waits for good.

``on_behalf`` is the protocol with a fault planted: a Q tile's stream does not look
at the K / V tiles it has no step for, and the other stream releases them for it.
"""

import random

import pytest


class Barrier:
    arrivals = 0                                          # of all barriers: something moves

    def __init__(self, count):
        self.count = self.pending = count
        self.done = 0

    def arrive(self):
        Barrier.arrivals += 1
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.done = self.count, self.done + 1

    def passed(self, parity):
        return (self.done & 1) != parity


class Stage:
    def __init__(self):
        self.full, self.empty, self.raw, self.tile = Barrier(1), Barrier(2), Barrier(1), None


class Model:
    """units: (end of Q tile 0, end of Q tile 1, V tiles at the end that the edge
    warp has to look at)."""

    def __init__(self, units, k_stages, v_stages, rng, on_behalf=False):
        self.units, self.rng, self.on_behalf = units, rng, on_behalf
        self.k = [Stage() for _ in range(k_stages)]
        self.v = [Stage() for _ in range(v_stages)]
        self.rows_look = v_stages == 1
        self.q_full, self.q_empty = [Barrier(1), Barrier(1)], [Barrier(1), Barrier(1)]
        self.s_full, self.o_full = [Barrier(1), Barrier(1)], [Barrier(1), Barrier(1)]
        self.p_full = [Barrier(1), Barrier(1)]
        self.work_full, self.work_empty = [Barrier(1), Barrier(1)], [Barrier(6), Barrier(6)]
        self.work = [None, None]
        self.flying, self.pipe, self.faults = [], [], []
        self.roles = [self.scheduler(), self.producer(), self.issuer(), self.rows(0), self.rows(1),
                      self.edge()]

    # ------------------------------------------------------------- the roles
    def scheduler(self):
        for c, unit in enumerate(self.units + [None]):
            while not self.work_empty[c & 1].passed(((c >> 1) & 1) ^ 1):
                yield
            self.work[c & 1] = unit
            self.work_full[c & 1].arrive()
            yield

    def next_work(self, c):
        while not self.work_full[c & 1].passed((c >> 1) & 1):
            yield
        unit = self.work[c & 1]
        self.work_empty[c & 1].arrive()
        return unit

    def producer(self):
        t = c = 0
        loaded = [0, 0]

        def load_q(x, unit):
            if unit[x] > 0:
                while not self.q_empty[x].passed((loaded[x] & 1) ^ 1):
                    yield
                self.flying.append((self.q_full[x], None, None))
                loaded[x] += 1

        def load(stages, name, raw=False):
            stage = stages[t % len(stages)]
            while not stage.empty.passed(((t // len(stages)) & 1) ^ 1):
                yield
            if stage.full.done != t // len(stages) or stage.empty.done != t // len(stages):
                self.faults.append(f"{name} {t} loaded out of turn")
            stage.tile = stage.looked = None
            self.flying.append((stage.raw if raw else stage.full, stage, t))
            yield

        while (unit := (yield from self.next_work(c))) is not None:
            c += 1
            n = max(unit[:2])
            if n > 0:
                yield from load_q(0, unit)
            for j in range(n):
                yield from load(self.k, "K")
                if j == 0:
                    yield from load_q(1, unit)
                yield from load(self.v, "V", not self.rows_look and j >= n - unit[2])
                t += 1

    def look(self, t, who):
        stage = self.v[t % len(self.v)]
        if stage.tile != t:
            self.faults.append(f"{who} looks at V {t}, there is {stage.tile}")
        stage.looked = t

    def rows(self, x):
        base = c = steps = outs = 0
        while (unit := (yield from self.next_work(c))) is not None:
            c += 1
            n = max(unit[:2])
            for j in range(unit[x]):
                while not self.s_full[x].passed(steps & 1):
                    yield
                yield
                if self.rows_look and j >= n - unit[2]:
                    while not self.v[0].full.passed((base + j) & 1):
                        yield
                    self.look(base + j, f"rows {x}")
                    yield
                self.p_full[x].arrive()
                steps += 1
            if unit[x] > 0:
                while not self.o_full[x].passed(outs & 1):
                    yield
                outs += 1
            base += n

    def edge(self):
        base = c = 0
        parity = [0] * len(self.v)
        while (unit := (yield from self.next_work(c))) is not None:
            c += 1
            n = max(unit[:2])
            for t in range(base + max(n - unit[2], 0), base + n):
                if self.rows_look:
                    break
                st = t % len(self.v)
                while not self.v[st].raw.passed(parity[st]):
                    yield
                parity[st] ^= 1
                self.look(t, "edge warp")
                yield
                self.v[st].full.arrive()
            base += n

    def issuer(self):
        streams = [dict(x=x, need="unit", unit=0, q=0, steps=0, g=0, k=0, v=0, i=0, left=0, n=0,
                        other=0) for x in range(2)]

        def landed(stages, t):
            return stages[t % len(stages)].full.passed((t // len(stages)) & 1)

        def release(stages, t, s):
            empty = stages[t % len(stages)].empty
            self.pipe.append(("arrive", empty))
            if self.on_behalf and s["i"] >= s["other"]:
                empty.arrive()

        def walk(s):
            for key, stages in (("k", self.k), ("v", self.v)):
                while s[key] < s["g"] and (key == "k" or s["v"] < s["k"]) and \
                        (self.on_behalf or landed(stages, s[key])):
                    if not self.on_behalf:
                        stages[s[key] % len(stages)].empty.arrive()
                    s[key] += 1

        def feed(s):
            x = s["x"]
            while s["need"] == "unit":
                slot = s["unit"] & 1
                if not self.work_full[slot].passed((s["unit"] >> 1) & 1):
                    break
                unit = self.work[slot]
                s["i"] = 0
                s["n"] = max(unit[:2]) if unit else 0
                s["left"] = unit[x] if unit else 0
                s["other"] = unit[x ^ 1] if unit else 0
                self.work_empty[slot].arrive()
                s["unit"] += 1
                s["need"] = "none" if unit is None else "qk" if s["left"] > 0 else "unit"
                if s["need"] == "unit":
                    s["g"] += s["n"]
            walk(s)
            if s["need"] == "qk":
                t = s["g"] + s["i"]
                if not self.on_behalf and (s["k"] < t or self.rows_look and s["v"] < t):
                    return
                if s["i"] == 0 and not self.q_full[x].passed(s["q"] & 1):
                    return
                if not landed(self.k, t):
                    return
                self.pipe += [("product", self.k, t, f"scores {x}"), ("arrive", self.s_full[x])]
                release(self.k, t, s)
                s["k"] = t + 1
                if s["i"] == s["left"] - 1:
                    self.pipe.append(("arrive", self.q_empty[x]))
                    s["q"] += 1
                s["need"] = "p"

        def serve(s):
            x, t = s["x"], s["g"] + s["i"]
            while not self.p_full[x].passed(s["steps"] & 1):
                yield
            unit = self.units[s["unit"] - 1]
            self.pipe.append(("edge product" if s["i"] >= max(unit[:2]) - unit[2] else "product",
                              self.v, t, f"values {x}"))
            s["steps"] += 1
            if s["i"] == s["left"] - 1:
                self.pipe.append(("arrive", self.o_full[x]))
            release(self.v, t, s)
            s["v"] = t + 1
            s["i"] += 1
            s["need"] = "qk" if s["i"] < s["left"] else "unit"
            if s["need"] == "unit":
                s["g"] += s["n"]
            feed(s)
            yield

        turn = 0
        while any(s["need"] != "none" for s in streams):
            w = [s["need"] == "p" and (self.on_behalf or s["v"] == s["g"] + s["i"]) and
                 landed(self.v, s["g"] + s["i"]) for s in streams]
            go = None
            for x in range(2):
                free = streams[x ^ 1]["need"] == "none" or \
                    self.p_full[x].passed(streams[x]["steps"] & 1)
                if go is None and w[x] and (turn == x if w[x ^ 1] else free):
                    go = x
            if go is not None:
                yield from serve(streams[go])
                turn = go ^ 1
            for s in streams:
                if s["need"] in ("unit", "qk"):
                    feed(s)
                elif s["v"] < s["g"]:
                    walk(s)
            yield

    # --------------------------------------------------------- the hardware
    def land(self):
        if not self.flying:
            return
        full, stage, tile = self.flying.pop(self.rng.randrange(len(self.flying)))
        if stage:
            stage.tile = tile
        full.arrive()

    def tensor(self):
        if not self.pipe:
            return
        op = self.pipe.pop(0)
        if op[0] == "arrive":
            op[1].arrive()
        elif op[1][op[2] % len(op[1])].tile != op[2] or \
                (op[0] == "edge product" and op[1][op[2] % len(op[1])].looked != op[2]):
            self.faults.append(f"{op[3]} of tile {op[2]} read {op[1][op[2] % len(op[1])].tile}")

    def run(self):
        """None when all roles end without a fault, else what went wrong."""
        actors = {i: r.__next__ for i, r in enumerate(self.roles)}
        roles = len(actors)
        weights = [self.rng.choice([1, 1, 10]) for _ in range(roles + 2)]
        weights[roles] = self.rng.choice([0.1, 1, 10])    # loads may be slow
        actors.update({roles: self.land, roles + 1: self.tensor})
        still, sweeps = set(), 0                          # polled since something moved
        while any(i in actors for i in range(roles)):
            i = self.rng.choices(list(actors), [weights[a] for a in actors])[0]
            before = (Barrier.arrivals, len(self.flying), len(self.pipe), len(actors))
            try:
                actors[i]()
            except StopIteration:
                del actors[i]
            if self.faults:
                return self.faults[0]
            moved = before != (Barrier.arrivals, len(self.flying), len(self.pipe), len(actors))
            still, sweeps = (set(), 0) if moved else (still | {i}, sweeps)
            if still == set(actors):
                still, sweeps = set(), sweeps + 1
            if sweeps == 4:
                return "deadlock"
        return None


PLANS = [(2, 1), (3, 2), (4, 4)]  # K and V stages at head sizes 192, 128 and 64


def units(rng):
    """Ends of the two Q tiles as the scheduler makes them: equal, one key tile
    apart, or one tile without a token (or without a key)."""
    made = []
    for _ in range(rng.randrange(1, 9)):
        n = rng.randrange(1, 7) if rng.random() < 0.6 else 1
        made.append(rng.choice([(n, n), (n - 1, n), (n - 1, n), (n, 0), (0, 0)]) +
                    (rng.randrange(4),))
    return made


@pytest.mark.parametrize("k_stages, v_stages", PLANS)
def test_every_product_meets_its_tile(k_stages, v_stages):
    for seed in range(250):
        rng = random.Random(seed)
        assert Model(units(rng), k_stages, v_stages, rng).run() is None, seed


@pytest.mark.parametrize("k_stages, v_stages", PLANS)
def test_model_sees_a_stream_that_skips_tiles(k_stages, v_stages):
    for seed in range(1500):
        rng = random.Random(seed)
        wrong = Model(units(rng), k_stages, v_stages, rng, on_behalf=True).run()
        if wrong:
            assert "read" in wrong or "looks" in wrong
            return
    assert False, "no order of events found the planted fault"
