"""A model of the roles and barriers of k_attend_packed (kernels_packed.cu), run with random interleavings.

Every role (two MMA warps, the TMA warp, the V scrub warp, two times four softmax warps) is a generator with the
kernel's waits in the kernel's order; the tensor core's and the TMA unit's completions come from queues of their own.  A
wait in the kernel sees only the parity of a barrier's phases, so the model also says which phase each wait means, and
checks that the parity never answers for another one: not early (the phase before the last is still wanted), not late
(a second phase went by unseen).  A run that stops with roles still waiting is a deadlock.

The items come from the schedule of drawn lengths (nkv_attend_schedule) and from draws of their own; whoever changes the
kernel's protocol changes it here as well.
"""
import ctypes as C
import random

import pytest

WARPS = 4  # softmax warps per half


class Fault(AssertionError):
    pass


class Bar:
    def __init__(self, name, count=1):
        self.name, self.count, self.pending, self.done = name, count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending < 0:
            raise Fault(f"{self.name}: an arrival too many")
        if self.pending == 0:
            self.done += 1
            self.pending = self.count


class Cta:
    """One CTA's run over its items: (steps of half 0, of half 1, history, rows of half 0, of half 1)."""

    def __init__(self, items, stages, history, rng, mended=True):
        self.items, self.N, self.history, self.rng, self.mended = items, stages, history, rng, mended
        two, ring = range(2), range(stages)
        self.S = [[Bar(f"scores {h}{b}") for b in two] for h in two]
        self.P = [[Bar(f"P {h}{b}", WARPS) for b in two] for h in two]
        self.PV = [[Bar(f"PV {h}{b}") for b in two] for h in two]  # [0] the last but one of an item, [1] the last
        self.Qf, self.Qe = [Bar(f"Q full {h}") for h in two], [Bar(f"Q free {h}") for h in two]
        self.Of = [Bar(f"O free {h}", WARPS) for h in two]
        self.H, self.Hr = [Bar(f"history {e}") for e in range(4)], [Bar(f"history read {e}", WARPS) for e in range(4)]
        self.Kf, self.Ke = [Bar(f"K full {s}") for s in ring], [Bar(f"K empty {s}", 2) for s in ring]
        self.Vf, self.Vc, self.Ve = ([Bar(f"V full {s}") for s in ring], [Bar(f"V clean {s}") for s in ring],
                                     [Bar(f"V empty {s}", 2) for s in ring])
        self.queues = [[], [], []]  # the MMA warps' commits, in order; the TMA unit's loads, in any

    # A wait is (barrier, parity the kernel passes, phase it means).
    @staticmethod
    def tiles(it):
        return (max(it[0], it[1]) + 1) // 2

    def mma(self, h):
        q, N = self.queues[h], self.N
        tiles = use0 = use1 = 0
        for i, it in enumerate(self.items):
            nh, n = it[h], self.tiles(it)

            def scores(u):
                q.append(self.S[h][u & 1])
                if u == nh - 1:
                    q.append(self.Qe[h])

            def pv(u):
                if u >= nh - 2:
                    q.append(self.PV[h][int(u == nh - 1)])

            yield self.Qf[h], i & 1, i
            if n > 0:
                yield self.Kf[tiles % N], (tiles // N) & 1, tiles // N
            for u in range(min(nh, 2)):
                scores(u)
            if nh == 0:
                q.append(self.Qe[h])
            if n > 0:
                q.append(self.Ke[tiles % N])
            if i > 0:
                yield self.Of[h], (i & 1) ^ 1, i - 1
            if nh == 0 and self.mended:
                q.append(self.PV[h][1])
            for t in range(n):
                u, x = 2 * t, tiles + t
                st, nx, more = x % N, (x + 1) % N, t + 1 < n
                yield self.Vc[st], (x // N) & 1, x // N
                if more:
                    yield self.Kf[nx], ((x + 1) // N) & 1, (x + 1) // N
                if u < nh:
                    yield self.P[h][0], (use0 + t) & 1, use0 + t
                    pv(u)
                if u + 2 < nh:
                    scores(u + 2)
                if u + 1 < nh:
                    yield self.P[h][1], (use1 + t) & 1, use1 + t
                    pv(u + 1)
                q.append(self.Ve[st])
                if u + 3 < nh:
                    scores(u + 3)
                if more:
                    q.append(self.Ke[nx])
            tiles += n
            use0 += (nh + 1) // 2
            use1 += nh // 2

    def tma(self):
        q, N, items = self.queues[2], self.N, self.items
        kt = vt = slots = histories = 0
        held, parity, uses = [0] * N, [0] * 4, [0] * 4

        def load_k():
            nonlocal kt
            st = kt % N
            if kt >= N:
                yield self.Ke[st], (kt // N - 1) & 1, kt // N - 1
            q.append(self.Kf[st])
            kt += 1

        def slot_free(st, what):
            had, held[st] = held[st], what
            if had == 1:
                last = (vt + N - 1 - st) // N - 1
                yield self.Ve[st], last & 1, last
            elif had:
                e = had - 2
                yield self.Hr[e], (parity[e] & 1) ^ 1, uses[e] - 1

        def load_v():
            nonlocal slots, vt
            st = slots % N
            yield from slot_free(st, 1)
            if st != vt % N:
                raise Fault("a V tile's stage is not its count modulo the ring")
            q.append(self.Vf[st])
            slots += 1
            vt += 1

        def load_q(i):
            for h in (0, 1):
                if i > 0:
                    yield self.Qe[h], (i - 1) & 1, i - 1
                q.append(self.Qf[h])

        if items:
            if self.tiles(items[0]):
                yield from load_k()
            yield from load_q(0)
        for i, it in enumerate(items):
            n = self.tiles(it)
            for t in range(n):
                yield from load_v()
                if t + 1 < n:
                    yield from load_k()
            if i + 1 < len(items):
                if self.tiles(items[i + 1]):
                    yield from load_k()
                yield from load_q(i + 1)
            if self.history and it[2]:
                for e in range(4):
                    st = slots % N
                    yield from slot_free(st, 2 + e)
                    parity[e] ^= 1
                    uses[e] += 1
                    q.append(self.H[e])
                    slots += 1
                histories += 1
        # nothing in flight at the end
        for x in range(max(0, kt - N), kt):
            yield self.Kf[x % N], (x // N) & 1, x // N
        for x in range(max(0, vt - N), vt):
            yield self.Vf[x % N], (x // N) & 1, x // N
        if items:
            for h in (0, 1):
                yield self.Qf[h], (len(items) - 1) & 1, len(items) - 1
        if histories:
            for e in range(4):
                yield self.H[e], (histories - 1) & 1, histories - 1

    def scrub(self):
        vt = 0
        for it in self.items:
            for _ in range(self.tiles(it)):
                st = vt % self.N
                yield self.Vf[st], (vt // self.N) & 1, vt // self.N
                self.Vc[st].arrive()
                vt += 1

    def softmax(self, h, w):
        bits = histories = last = before_last = 0
        seen = [0, 0]  # phases of the score buffers
        for it in self.items:
            nh, idle = it[h], 32 * w >= it[3 + h]
            moves = [self.rng.random() < 0.3 for _ in range(nh)]  # the running maximum moves: O is rescaled
            waited = False

            def full(u):
                return self.S[h][u & 1], ((bits >> (u & 1)) ^ (u >> 1)) & 1, seen[u & 1] + (u >> 1)

            if not idle and nh:
                yield full(0)
            for u in range(nh):
                if idle:
                    yield full(u)
                elif u + 1 < nh:
                    yield full(u + 1)
                elif u > 0 and moves[u]:
                    yield self.PV[h][0], (bits >> 3) & 1, before_last
                    waited = True
                self.P[h][u & 1].arrive()
            bits ^= ((nh + 1) // 2) & 1
            bits ^= ((nh // 2) & 1) << 1
            seen[0] += (nh + 1) // 2
            seen[1] += nh // 2
            if nh > 0 or self.mended:
                if nh >= 2 and not waited:
                    yield self.PV[h][0], (bits >> 3) & 1, before_last
                yield self.PV[h][1], (bits >> 2) & 1, last
                bits ^= 12 if nh > 1 else 4
                last += 1
                before_last += nh > 1
            for e in (0, 1):  # the output's columns
                if e == 1:
                    self.Of[h].arrive()
                if self.history and it[2]:
                    yield self.H[2 * h + e], (bits >> 4) & 1, histories
                    self.Hr[2 * h + e].arrive()
            if self.history and it[2]:
                bits ^= 16
                histories += 1

    def run(self):
        rng = self.rng
        roles = {"tma": self.tma(), "scrub": self.scrub()}
        for h in (0, 1):
            roles[f"mma {h}"] = self.mma(h)
            for w in range(WARPS):
                roles[f"softmax {h}{w}"] = self.softmax(h, w)
        waiting = {}

        def step(name):
            try:
                waiting[name] = next(roles[name])
            except StopIteration:
                waiting.pop(name, None)
                del roles[name]

        for name in list(roles):
            step(name)
        speed = {name: rng.choice([0.02, 0.3, 1, 1, 1]) for name in roles}
        unit = [rng.choice([0.05, 0.5, 1]) for _ in self.queues]
        still = 0
        while roles:
            acted = False
            for k, q in enumerate(self.queues):
                if q and rng.random() < unit[k]:
                    q.pop(0 if k < 2 else rng.randrange(len(q))).arrive()
                    acted = True
            for name in rng.sample(list(waiting), len(waiting)):
                bar, parity, phase = waiting[name]
                if parity != phase & 1:
                    raise Fault(f"{name} passes parity {parity} for phase {phase} of {bar.name}")
                if (bar.done & 1) != parity:
                    if bar.done != phase + 1:
                        raise Fault(f"{name}: {bar.name} is at {bar.done}, answers for phase {phase}")
                    acted = True
                    if rng.random() < speed[name]:
                        step(name)
                elif bar.done > phase:
                    raise Fault(f"{name}: {bar.name} is at {bar.done}, phase {phase} went by")
            still = 0 if acted or any(self.queues) else still + 1
            if still > 50:
                raise Fault(f"deadlock: { {n: (w[0].name, w[2], w[0].done) for n, w in waiting.items()} }")


def _drawn(rng):
    items = []
    for _ in range(rng.choice([1, 2, 3, 5, 9])):
        n0 = rng.choice([1, 2, 3, 4, 7, 8])
        n1 = rng.choice([n0, n0 + 1, n0 + 2, n0 + 4])
        s0, s1 = rng.choice([(0, 0), (n0, 0), (n0, n1), (n0, n1), (0, n1)])
        items.append((s0, s1, rng.random() < 0.8, rng.choice([1, 40, 128]), rng.choice([0, 1, 128])))
    return items


def _scheduled(nkv, rng):
    """Items of a drawn plan: the steps that set_steps gives them."""
    n = rng.randint(1, 5)
    q = [rng.choice([0, 1, 3, rng.randint(1, 700)]) for _ in range(n)]
    k = [rng.choice([0, a, a + rng.randint(0, 2500), rng.randint(0, 300)]) for a in q]
    kv, G = rng.choice([1, 2]), rng.choice([1, 3, 8, 100])
    causal, block = rng.randint(0, 1), rng.choice([1, 100])
    qa, ka, cnt = (C.c_uint64 * n)(*q), (C.c_uint64 * n)(*k), C.c_uint64()
    args = (qa, ka, n, kv * G, kv, causal, block, rng.choice([1, 3, 20]))
    nkv._check(nkv.lib().nkv_attend_schedule(*args, None, 0, C.byref(cnt)))
    buf = (C.c_int64 * (8 * max(cnt.value, 1)))()
    nkv._check(nkv.lib().nkv_attend_schedule(*args, buf, cnt.value, C.byref(cnt)))
    starts, q0, k0 = {}, 0, 0
    for ql, kl in zip(q, k):
        if ql:
            starts[(q0, k0)] = (ql, kl)
        q0, k0 = q0 + ql, k0 + kl
    half = G * (128 // G)
    items = []
    for c in range(cnt.value):
        qs, ks, row0, rows, _, lo, hi, part = buf[8 * c:8 * c + 8]
        ql, kl = starts[(qs, ks)]

        def limit(row):
            p = row // G + kl - ql
            return kl if not causal else 0 if p < 0 else min(kl, (p // block + 1) * block)

        def steps(first, count):
            if count <= 0:
                return 0
            return max(0, -(-(min(limit(row0 + first + count - 1), 128 * hi) - 128 * lo) // 64))

        items.append((steps(0, min(half, rows)), steps(half, rows - half), part < 0, min(half, rows),
                      max(0, rows - half)))
    at = rng.randrange(max(1, len(items)))
    return items[at:at + rng.choice([1, 3, 8])]  # some CTA's run of them


@pytest.mark.parametrize("stages", [2, 4])
@pytest.mark.parametrize("seed", range(4))
def test_every_wait_gets_the_phase_it_means(nkv, seed, stages):
    rng = random.Random(100 * stages + seed)
    for i in range(40):
        items = _scheduled(nkv, rng) if i % 2 else _drawn(rng)
        Cta(items, stages, rng.random() < 0.5, rng).run()


def test_the_model_finds_a_missing_phase():
    """Without the "last PV" of a half that has no steps, its softmax warps free O twice before the wait for the first."""
    found = 0
    for seed in range(120):
        rng = random.Random(seed)
        items, stages, history = _drawn(rng), rng.choice([2, 4]), rng.random() < 0.5
        try:
            Cta(items, stages, history, rng, mended=False).run()
        except Fault:
            found += 1
    assert found >= 12
