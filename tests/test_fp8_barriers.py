"""The barrier protocols of the 8-bit products (csrc/gemm_fp8.cu), run on the CPU many times with their roles, copies and MMAs in random order.  Barriers know
phases and parities alone, as the hardware's do; what lies in stages, factor slots and tensor memory is tracked by block: whoever reads finds the block that it
is about, nothing is written that is still to be read, and nobody waits for ever."""
import os
import random
import re

import pytest

SRC = open(os.path.join(os.path.dirname(__file__), "..", "kubernetes-gpu-cluster_b200", "csrc", "gemm_fp8.cu")).read()

# every barrier operation of the roles, in the order of the source: what the programs below transcribe
STREAM_OPS = [
    "expect full(ahead), bytes_of(t, n)", "wait empty(stage), phase ^ 1", "expect full(stage), bytes_of(t, n)",
    "wait full(stage), phase", "wait tempty(buf), buf_phase ^ 1", "test full(s1), p1", "test tempty(v1), w1 ^ 1", "commit tfull(buf)", "commit empty(stage)",
    "wait empty(stage), phase ^ 1",
    "arrive tempty(buf)", "wait tfull(buf), buf_phase", "wait tfull(buf), buf_phase"]
PAIR_OPS = [
    "wait empty(stage), phase ^ 1", "expect full(stage), 2 * kStage", "arrive lead",
    "wait full(stage), phase", "wait tempty(2 * buf + h), buf_phase ^ 1", "test full(s1), p1", "test tempty(2 * v1 + h), w1 ^ 1", "commit tfull(2 * buf + h), 3",
    "commit empty(stage), 3",
    "wait tfull(2 * buf + part), buf_phase", "arrive lead_tempty + 16u * buf", "wait tfull(2 * buf + part), buf_phase", "wait tfull(2 * buf + part), buf_phase"]
CALLS = {"mbar_wait": "wait", "mbar_test": "test", "bar_expect": "expect", "bar_arrive": "arrive", "bar_arrive_at": "arrive", "bar_arrive_lane0": "arrive", "commit": "commit", "commit2": "commit"}


def operations(kernel, begin):
    body = SRC[SRC.index(kernel + "(const __grid"):]
    body = body[body.index(begin):]
    body = re.sub(r"//[^\n]*", "", body[:re.search(r"\n}\n", body).start()])
    out = []
    for m in re.finditer(r"\b(" + "|".join(CALLS) + r")\(", body):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(body[i], 0)
            i += 1
        out.append(CALLS[m.group(1)] + " " + body[m.end():i - 1].removesuffix(", lane"))
    return out


def constant(name):
    return int(re.search(r"\b%s = (\d+)\b" % name, SRC).group(1))


def test_transcriptions_match_the_kernels():
    assert operations("fp8_stream_kernel", "  if (warp == 0) {\n    regs_down") == STREAM_OPS
    assert operations("fp8_pair_kernel", "  if (warp == 0 || warp == 3) {") == PAIR_OPS
    assert constant("kPairStages") > constant("kPairBatch") and "kPairSlots = kPairStages + 2;" in SRC and "slots = (stages + BUFS) * SUB;" in SRC
    for count in ("bar_init(full(s), 33); bar_init(empty(s), 1);", "bar_init(tfull(b), 1); bar_init(tempty(b), kSumWarps);", "bar_init(full(s), 3); bar_init(empty(s), 2);"):
        assert count in SRC


class Barrier:
    def __init__(self, need):
        self.need, self.got, self.done = need, 0, 0

    def arrive(self):
        self.got += 1
        assert self.got <= self.need
        if self.got == self.need:
            self.got, self.done = 0, self.done + 1

    def passed(self, parity):                             # of a phase that the caller names by its parity
        return (self.done & 1) != (parity & 1)


def run(roles, flights, rng):
    """Roles are generators that yield a condition to wait for (or None); flights: functions that return what may complete now (lists of callables)."""
    waiting = [next(r, "end") for r in roles]
    quiet = 0
    while any(w != "end" for w in waiting):
        ready = [("role", i) for i, w in enumerate(waiting) if w != "end" and (w is None or w())]
        ready += [("flight", f) for group in flights for f in group()]
        assert ready, "waits for ever"
        kind, what = rng.choice(ready)
        if kind == "role":
            waiting[what] = next(roles[what], "end")
        else:
            what()
        quiet += 1
        assert quiet < 100000


class Copies:
    """Copies in flight: any of them may arrive next."""

    def __init__(self):
        self.todo = []

    def start(self, fn):
        self.todo.append(fn)

    def ready(self):
        def take(fn):
            self.todo.remove(fn)
            fn()
        return [lambda fn=fn: take(fn) for fn in self.todo]


class Tensor(Copies):
    """MMAs complete in the order of issue."""

    def ready(self):
        return super().ready()[:1]


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("tiles,KB", [(1, 1), (1, 7), (5, 1), (4, 2), (3, 5), (2, 11), (3, 16)])
def test_pairs(seed, tiles, KB):
    """Two CTAs: two producers and two groups of sums each, two threads that issue."""
    S, BATCH = constant("kPairStages"), constant("kPairBatch")
    SLOTS, rng = S + 2, random.Random(seed * 1000 + tiles * 50 + KB)
    full = [Barrier(3 + 2) for _ in range(S)]             # (and both CTAs' copies, which the hardware counts in bytes)
    empty = [[Barrier(2) for _ in range(S)] for _ in range(2)]
    tfull = [[Barrier(1) for _ in range(4)] for _ in range(2)]
    tempty = [Barrier(4) for _ in range(4)]               # (two groups of two CTAs; a group's four warps here in two halves)
    stage_of, factor, acc, info = [[None] * S for _ in range(2)], [[None] * SLOTS for _ in range(2)], [None] * 4, [[None] * 16 for _ in range(2)]
    copies, tensor, left = Copies(), Tensor(), {}
    total = tiles * KB

    def producer(cta, warp):
        stage, slot, phase, turn = 0, 0, 0, 1 - warp
        for tile in range(tiles):
            if turn:
                info[cta][tile & 15] = tile
            for kb in range(0, KB, BATCH):
                n = min(BATCH, KB - kb)
                turn ^= 1
                if turn:
                    stage += n
                    while stage >= S:
                        stage, phase = stage - S, phase ^ 1
                    slot = (slot + n) % SLOTS
                    continue
                for i in range(n):
                    block = tile * KB + kb + i
                    b, p = empty[cta][stage], phase ^ 1
                    yield lambda b=b, p=p: b.passed(p)
                    assert b.done >= block // S, "the stage is not free"
                    if cta == 0:
                        full[stage].arrive()

                    def land(stage=stage, block=block):
                        assert left.get(("stage", cta, stage), 0) == 0, "a stage is overwritten"
                        stage_of[cta][stage] = block
                        left[("stage", cta, stage)] = 2
                        full[stage].arrive()
                    copies.start(land)
                    yield None
                    assert left.get(("factor", cta, slot), 0) == 0, "factors are overwritten"
                    factor[cta][slot] = block
                    left[("factor", cta, slot)] = 4
                    full[stage].arrive()
                    yield None
                    stage, phase = (0, phase ^ 1) if stage + 1 == S else (stage + 1, phase)
                    slot = (slot + 1) % SLOTS

    def issuer(h):
        stage, buf, phase, buf_phase, f_there, t_there = 0, 0, 0, 0, False, False
        for block in range(total):
            if not f_there:
                yield lambda: full[stage].passed(phase)
            if not t_there:
                yield lambda: tempty[2 * buf + h].passed(buf_phase ^ 1)
            assert full[stage].done == block // S + 1 and tempty[2 * buf + h].done == block // 2
            s1, v1 = (stage + 1) % S, buf ^ 1
            p1, w1 = phase ^ (s1 == 0), buf_phase ^ buf
            f_there, t_there = full[s1].passed(p1), tempty[2 * v1 + h].passed(w1 ^ 1)
            yield None

            def mma(stage=stage, buf=buf, block=block):
                for cta in range(2):
                    assert stage_of[cta][stage] == block
                    left[("stage", cta, stage)] -= 1
                assert left.get(("acc", 2 * buf + h), 0) == 0, "sums are overwritten"
                acc[2 * buf + h] = block
                left[("acc", 2 * buf + h)] = 4
                for cta in range(2):
                    tfull[cta][2 * buf + h].arrive()
                    empty[cta][stage].arrive()
            tensor.start(mma)
            yield None
            stage, phase, buf, buf_phase = s1, p1, v1, w1

    def sums(cta, part):
        buf, slot, buf_phase = 0, 0, 0
        for block in range(total):
            yield lambda: tfull[cta][2 * buf + part].passed(buf_phase)
            assert info[cta][block // KB & 15] == block // KB and factor[cta][slot] == block and acc[2 * buf + part] == block
            yield None
            left[("factor", cta, slot)] -= 1
            left[("acc", 2 * buf + part)] -= 1
            tempty[2 * buf + part].arrive()
            buf, buf_phase = buf ^ 1, buf_phase ^ buf
            slot = (slot + 1) % SLOTS
    roles = [producer(c, w) for c in range(2) for w in range(2)] + [issuer(h) for h in range(2)] + [sums(c, p) for c in range(2) for p in range(2) for _ in range(2)]
    run(roles, [copies.ready, tensor.ready], rng)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("stages,sub", [(2, 1), (3, 1), (5, 1), (2, 2), (3, 2), (8, 2)])
@pytest.mark.parametrize("tiles,KB,ahead", [(1, 1, 1), (1, 9, 2), (1, 16, 8), (3, 5, 0), (4, 3, 2), (5, 8, 0)])
def test_single_ctas(seed, stages, sub, tiles, KB, ahead):
    """A producer (whose first tile's weights are under way early), a warp that copies factors, an issuing thread, groups of sums."""
    rng = random.Random(seed * 1000 + stages * 100 + tiles * 10 + KB)
    bufs, slots = 2, (stages + 2) * sub
    full, empty = [Barrier(3) for _ in range(stages)], [Barrier(1) for _ in range(stages)]      # (full: the producer, its copies, the factors' copies)
    tfull, tempty = [Barrier(1) for _ in range(bufs)], [Barrier(2) for _ in range(bufs)]
    held, factor, acc, left = [None] * stages, [None] * slots, [None] * bufs, {}
    copies, tensor = Copies(), Tensor()
    steps = [(t, kb, min(sub, KB - kb)) for t in range(tiles) for kb in range(0, KB, sub)]
    per = -(-KB // sub)

    def land(stage, n):
        def fn():
            assert left.get(("stage", stage), 0) == 0, "a stage is overwritten"
            held[stage] = n
            left[("stage", stage)] = 1
            full[stage].arrive()
        return fn

    def producer():
        early = min(ahead, stages, per)
        for n in range(early):
            full[n].arrive()
        stage, phase = 0, 0
        yield None
        for n in range(len(steps)):
            if n >= early:
                yield lambda: empty[stage].passed(phase ^ 1)
                full[stage].arrive()
            copies.start(land(stage, n))
            yield None
            stage, phase = (0, phase ^ 1) if stage + 1 == stages else (stage + 1, phase)

    def helper():
        stage, phase, slot = 0, 0, 0
        for n, (_, _, k) in enumerate(steps):
            yield lambda: empty[stage].passed(phase ^ 1)
            assert empty[stage].done >= n // stages

            def fn(n=n, k=k, slot=slot, stage=stage):
                for u in range(k):
                    assert left.get(("factor", slot + u), 0) == 0, "factors are overwritten"
                    factor[slot + u] = (n, u)
                    left[("factor", slot + u)] = 2
                full[stage].arrive()
            copies.start(fn)
            yield None
            stage, phase = (0, phase ^ 1) if stage + 1 == stages else (stage + 1, phase)
            slot = (slot + sub) % slots

    def issuer():
        stage, buf, phase, buf_phase, f_there, t_there = 0, 0, 0, 0, False, False
        for n in range(len(steps)):
            if not f_there:
                yield lambda: full[stage].passed(phase)
            if not t_there:
                yield lambda: tempty[buf].passed(buf_phase ^ 1)
            assert full[stage].done == n // stages + 1 and tempty[buf].done == n // bufs
            s1, v1 = (stage + 1) % stages, (buf + 1) % bufs
            p1, w1 = phase ^ (s1 == 0), buf_phase ^ (v1 == 0)
            f_there, t_there = full[s1].passed(p1), tempty[v1].passed(w1 ^ 1)
            yield None

            def mma(stage=stage, buf=buf, n=n):
                assert held[stage] == n and left.get(("acc", buf), 0) == 0
                left[("stage", stage)] -= 1
                acc[buf], left[("acc", buf)] = n, 2
                tfull[buf].arrive()
                empty[stage].arrive()
            tensor.start(mma)
            yield None
            stage, phase, buf, buf_phase = s1, p1, v1, w1

    def sums():
        buf, slot, buf_phase, at = 0, 0, 0, 0
        for n, (t, kb, k) in enumerate(steps):
            yield lambda: tfull[buf].passed(buf_phase)
            for u in range(k):
                assert acc[buf] == n and factor[slot + u] == (n, u)
                yield None
                left[("factor", slot + u)] -= 1
            left[("acc", buf)] -= 1
            tempty[buf].arrive()
            buf, buf_phase = (0, buf_phase ^ 1) if buf + 1 == bufs else (buf + 1, buf_phase)
            slot = (slot + sub) % slots
    run([producer(), helper(), issuer(), sums(), sums()], [copies.ready, tensor.ready], rng)


def test_registers_add_up():
    """What the groups take on and give up is no more than the block is launched with."""
    threads, sums, others = 384, constant("kSumRegs"), constant("kOtherRegs")
    launched = 65536 // threads // 8 * 8
    assert 256 * sums + 128 * others <= threads * launched and sums <= 232


class Telling(Barrier):
    """A barrier of one CTA that passes on what those who arrive know, to waiters of their own CTA: arrivals and waits without a scope are of the CTA."""

    def __init__(self, need):
        super().__init__(need)
        self.known = {0: set(), 1: set()}

    def arrive(self, cta=None, knows=()):
        if cta is not None:
            self.known[cta] |= set(knows)
        super().arrive()


def pairs_with_scopes(seed, tiles, KB, told_by_slot):
    """The pair kernel's way of the factors alone: written by a CTA's producers, read by its sums; the leader's issuing thread is in between, or a slot's own barrier."""
    S, BATCH, total = constant("kPairStages"), constant("kPairBatch"), tiles * KB
    SLOTS, rng = S + 2, random.Random(seed)
    full, empty = [Telling(3) for _ in range(S)], [[Telling(1) for _ in range(S)] for _ in range(2)]
    tfull, tempty = [[Telling(1) for _ in range(2)] for _ in range(2)], [Telling(2) for _ in range(2)]
    told = [[Telling(1) for _ in range(SLOTS)] for _ in range(2)]
    order = [tile * KB + kb for tile in range(tiles) for kb in range(KB)]
    turn_of = {tile * KB + kb: kb // BATCH % 2 for tile in range(tiles) for kb in range(KB)}

    def producer(cta, warp):
        knows = set()
        for b in order:
            if turn_of[b] != warp:
                continue
            yield lambda: empty[cta][b % S].passed(b // S & 1 ^ 1)
            if cta == 0:
                full[b % S].arrive()
            knows.add(b)                                      # (the slot's factors, and the tile's place with its first)
            yield None
            told[cta][b % SLOTS].arrive(cta, knows)
            full[b % S].arrive(cta, knows)
            yield None

    def issuer():
        knows = set()
        for b in order:
            yield lambda: full[b % S].passed(b // S & 1)
            knows |= full[b % S].known[0]
            yield lambda: tempty[b % 2].passed(b // 2 & 1 ^ 1)
            for cta in range(2):
                tfull[cta][b % 2].arrive(0, knows)
                empty[cta][b % S].arrive(0, knows)
            yield None

    def sums(cta):
        knows, seen = set(), False
        for b in order:
            if told_by_slot:
                if not seen:
                    yield lambda: told[cta][b % SLOTS].passed(b // SLOTS & 1)
                assert told[cta][b % SLOTS].done == b // SLOTS + 1
                knows |= told[cta][b % SLOTS].known[cta]
                seen = told[cta][(b + 1) % SLOTS].passed((b + 1) // SLOTS & 1) and b + 1 < total
            yield lambda: tfull[cta][b % 2].passed(b // 2 & 1)
            knows |= tfull[cta][b % 2].known[cta]
            assert b in knows, "factors are read that nobody has published"
            tempty[b % 2].arrive(cta, knows)
            yield None
    run([producer(c, w) for c in range(2) for w in range(2)] + [issuer(), sums(0), sums(1)], [], rng)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("tiles,KB", [(1, 1), (1, 7), (5, 1), (4, 2), (3, 5), (2, 11), (2, 24)])
def test_factors_are_published_within_their_cta(seed, tiles, KB):
    pairs_with_scopes(seed, tiles, KB, True)
    with pytest.raises(AssertionError, match="nobody has published"):      # by way of the leader alone the second CTA's are not
        pairs_with_scopes(seed, tiles, KB, False)


def test_a_slot_is_told_before_it_is_read():
    """In the source: a producer tells a slot behind its factors, readers wait for it before the tile's place and before every block's factors."""
    body = re.sub(r"//[^\n]*", "", SRC[SRC.index("fp8_pair_kernel(const __grid"):])
    assert re.search(r"f\.put\(factors \+ slot \* 256, i, lane\);\s*__syncwarp\(\);\s*if \(lane == 0\) \{\s*told\.tell\(slot\);", body)
    assert re.search(r"told\.wait\(slot, slot_phase\);\s*mbar_wait\(tfull\(2 \* buf \+ part\), buf_phase\);\s*const int4 found = tiles", body)
    assert re.search(r"if \(!seen\) told\.wait\(slot, slot_phase\);\s*const bool last = [^;]*;\s*seen = told\.test\([^;]*;\s*const float\* f = factors", body)
    assert body.count("= factors + slot") == 1 and body.count("= tiles[") == 1


@pytest.mark.parametrize("kernel,roles", [("fp8_stream_kernel", 4), ("fp8_pair_kernel", 3)])
def test_no_barrier_wait_spans_the_kernel_before(kernel, roles):
    """Waits at barriers are limited in time, and what the kernel before takes is not: whoever waits at one has waited for that kernel's end first."""
    body = re.sub(r"//[^\n]*", "", SRC[SRC.index(kernel + "(const __grid"):])
    body = body[:re.search(r"\n}\n", body).start()]
    parts = re.split(r"\n  (?:\} else )?(?:if \(warp [^\n]*\) \{|else \{|\} else \{)\s*\n    regs_\w+<\w+>\(\);", body)
    begin, waiting = parts[0], [r for r in parts[1:] if re.search(r"\bmbar_wait\(|\.wait\(", r)]
    assert len(waiting) == roles and "mbar_wait(" not in begin
    for role in waiting:
        assert re.search(r"\n  pdl_wait\(\);", begin) or role.index("pdl_wait();") < re.search(r"\bmbar_wait\(|\.wait\(", role).start()


def exchange(S, over, gated, rng, early=False):
    """The end of a cluster's tile (fp8_stream_kernel, CLUSTER): S CTAs, in each the warps that add up and the others, who take the same barriers of the cluster."""
    arrived, counts = [0] * 8, {}                             # phases of the cluster's barrier: two arrivals a CTA each
    stages_read, begun, gone = [False] * S, [False] * S, [0] * S
    sums, tops, kept = [set() for _ in range(S)], [set() for _ in range(S)], [False] * S

    def arrive(who):
        arrived[counts.setdefault(who, 0)] += 1
        counts[who] += 1

    def wait(who):
        return lambda: arrived[counts[who] - 1] == 2 * S

    def remote(c):
        assert begun[c], "a CTA that may not have begun is written to"
        assert gone[c] < 2, "a CTA that may be gone is written to"

    def adding(c):
        me = ("sums", c)
        yield None
        begun[c] = True
        if not over:
            arrive(me)
        yield None
        stages_read[c] = True                                  # (its last block's sums are there: the MMAs have read the stages)
        if over and not early:
            arrive(me)
        if not early:
            yield wait(me)
        for to in range(S):
            remote(to)
            assert not over or stages_read[to], "sums are laid over stages that are still read"
            assert c not in sums[to]
            sums[to].add(c)
            yield None
        arrive(me)
        yield wait(me)
        assert len(sums[c]) == S, "sums are missing"
        if gated:
            kept[c] = True                                     # (h, in the place of the first sender's sums)
            for to in range(S):
                remote(to)
                tops[to].add(c)
                yield None
            arrive(me)
            yield wait(me)
            assert len(tops[c]) == S and kept[c]
        gone[c] += 1

    def others(c):
        me = ("others", c)
        yield None
        if not over:
            arrive(me)
        yield None
        for n in range(1 + (over and not early) + gated):
            if n == 0 and not over:
                yield wait(me)
            arrive(me)
            yield wait(me)
        gone[c] += 1
    run([r for c in range(S) for r in (adding(c), others(c))], [], rng)
    assert all(len(s) == S for s in sums) and len(set(counts.values())) == 1


@pytest.mark.parametrize("S", [2, 3, 5, 8])
@pytest.mark.parametrize("over,gated", [(False, False), (False, True), (True, True)])
def test_a_clusters_exchange(S, over, gated):
    for seed in range(40):
        exchange(S, over, gated, random.Random(seed * 10 + S))


def test_an_exchange_without_its_first_barrier_is_seen():
    with pytest.raises(AssertionError, match="begun|still read"):
        for seed in range(40):
            exchange(4, True, True, random.Random(seed), early=True)


def test_all_warps_take_the_clusters_barriers_alike():
    """In the source: before the roles, by those that add up, and by the others behind them."""
    body = re.sub(r"//[^\n]*", "", SRC[SRC.index("fp8_stream_kernel(const __grid"):])
    body = body[:re.search(r"\n}\n", body).start()]
    calls = re.findall(r"(?:if \([^()]*\) )?\{? ?cluster_(?:arrive_relaxed|arrive|wait)\(\);", body)
    take = lambda part: ["over: arrive" if "p.over" in c and "arrive()" in c else re.search(r"arrive_relaxed|arrive|wait", c).group() for c in part]
    assert "CLUSTER && !p.over" in calls[0] and take(calls) == ["arrive_relaxed"] + 2 * ["over: arrive", "wait", "arrive", "wait", "arrive", "wait"]
    assert body.count("if constexpr (GATED) {\n          // the block's largest") <= 1 and "if (GATED) { cluster_arrive(); cluster_wait(); }" in body
