"""The barrier protocols of attention over the 4-bit cache, explored on the CPU over every order in which their roles can run: the prompt kernel
(csrc/attn_kv4_tc.cuh), where warps of their own turn codes into tiles, and the ring of shares of long contexts (csrc/attn_kv4.cu).  No wait may
be left behind by its barrier, none may pass early, and no buffer may be overwritten before its readers are done."""
import os
import re

import pytest

import barrier_explorer

CSRC = os.path.join(os.path.dirname(__file__), "..", "kubernetes-gpu-cluster_b200", "csrc")

# every barrier operation behind the barriers' set-up, in the order of the source: what the programs below transcribe
PROMPT_OPS = [
    # producer
    "wait item_empty(slot), ((ni >> 1) - 1) & 1", "arrive item_full(slot)", "wait q_empty, (ni - 1) & 1", "wait raw_empty(st), (nraw / NRAW - 1) & 1",
    "wait clc_full, nclc & 1", "wait item_empty(slot), ((ni >> 1) - 1) & 1", "arrive item_full(slot)",
    # issuers
    "wait item_full(ni & 1), (ni >> 1) & 1", "arrive item_empty(ni & 1)", "wait q_full, ni & 1",
    "wait k_full(st), ((nk + js) / NST) & 1", "wait s_read(a), (ns - 1) & 1", "commit s_full(a)", "commit k_empty(st)", "commit q_empty",
    "wait v_full(st), ((nk + j) / NST) & 1", "wait p_full(a, np), (np >> 1) & 1", "commit o_full(a, np)", "commit v_empty(st)",
    # turning warps
    "wait item_full(ni & 1), (ni >> 1) & 1", "arrive item_empty(ni & 1)", "wait raw_full(rs), (nk / NRAW) & 1",
    "wait part_v ? v_empty(st) : k_empty(st), (nk / NST - 1) & 1", "arrive part_v ? v_full(st) : k_full(st)", "arrive raw_empty(rs)",
    # softmax warps
    "wait item_full(ni & 1), (ni >> 1) & 1", "arrive item_empty(ni & 1)", "wait q_full, ni & 1", "arrive q_empty", "wait s_full(a), ns & 1", "arrive s_read(a)",
    "wait v_full(st), ((nk + jt) / NST) & 1", "wait o_full(a, ns - 1), ((ns - 1) >> 1) & 1", "wait o_full(a, ns), ((ns - 2) >> 1) & 1", "arrive p_full(a, ns)",
    "wait o_full(a, ns - 1), ((ns - 1) >> 1) & 1",
]
SHARE_OPS = [
    # producer
    "idle p_empty(pi), p_parity ^ 1", "expect p_full(pi), (uint32_t)(G * HD * 2)", "idle empty(stage), parity ^ 1", "expect full(stage), bytes",
    "idle p_empty(pi), p_parity ^ 1", "arrive p_full(pi)",
    # computing warps
    "wait p_full(pi), p_parity", "arrive p_empty(pi)", "wait full(stage), parity", "arrive empty(stage)",
]


def barrier_ops(name, begin, end, calls):
    src = open(os.path.join(CSRC, name)).read()
    body = src[src.index(begin):]
    body = re.sub(r"//[^\n]*", "", body[:body.index(end)])
    out = []
    for m in re.finditer(r"\b(" + "|".join(calls) + r")\(", body):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(body[i], 0)
            i += 1
        out.append(calls[m.group(1)] + " " + body[m.end():i - 1])
    return out


def test_transcriptions_match_the_kernels():
    assert barrier_ops("attn_kv4_tc.cuh", "if (warp == 10) {\n", "}  // namespace atc4", {"mbar_wait": "wait", "mbar_arrive": "arrive", "tc_commit": "commit"}) == PROMPT_OPS
    assert barrier_ops("attn_kv4.cu", "    int4 desc = make_int4(-1, 0, 0, 0);", "// Groups that were cut",
                       {"mbar_wait_idle": "idle", "mbar_wait": "wait", "mbar_arrive": "arrive", "mbar_expect": "expect"}) == SHARE_OPS


# --------------------------------------------------------------------------------------------------------------- prompts

def wait(bar, k, optional=False):
    return ("maybe" if optional else "wait", bar, k)


def programs(items, nst, nraw, turners):
    """Instruction lists of the roles: producer, two issuers, the turning warps, two groups of softmax warps.  items: (key tiles of the first
    query tile, of the second[, whether they share the key tiles of one query tile between them])."""
    prod, nk, end = [], 0, len(items)
    items = [(*i, 0)[:3] for i in items]
    tiles = [i[0] + i[1] if i[2] else max(i[:2]) for i in items]
    for ni in range(end + 1):
        if ni >= 2:
            prod.append(wait(("item_empty", ni & 1), (ni >> 1) - 1))
        prod.append(("arrive", ("item_full", ni & 1)))
        if ni == end:
            break
        if ni:
            prod.append(wait(("q_empty",), ni - 1))
        prod.append(("load", ("q_full",), ("q",)))
        for _ in range(tiles[ni]):
            if nk >= nraw:
                prod.append(wait(("raw_empty", nk % nraw), nk // nraw - 1))
            prod.append(("load", ("raw_full", nk % nraw), ("raw", nk % nraw)))
            nk += 1
    roles = [prod]
    for a in range(2):
        issue, ns, np, nk = [], 0, 0, 0
        for ni, nn in enumerate(items):
            n, ahead = tiles[ni], 1 + nn[2]
            issue += [wait(("item_full", ni & 1), ni >> 1), ("arrive", ("item_empty", ni & 1)), wait(("q_full",), ni)]
            for j in range(-ahead, n):
                js = j + ahead
                if js < n:
                    st = (nk + js) % nst
                    issue.append(wait(("k_full", st), (nk + js) // nst))
                    if js % 2 == a if nn[2] else js < nn[a]:
                        if ns:
                            issue.append(wait(("s_read", a), ns - 1))
                        issue.append(("mma", [("s_full", a)], [("q",), ("k", st)], [("s", a)]))
                        ns += 1
                    issue.append(("mma", [("k_empty", st)] + ([("q_empty",)] if js + 1 == n else []), [], []))
                if j >= 0:
                    st = (nk + j) % nst
                    issue.append(wait(("v_full", st), (nk + j) // nst))
                    if j % 2 == a if nn[2] else j < nn[a]:
                        issue += [wait(("p_full", a, np & 1), np >> 1), ("mma", [("o_full", a, np & 1)], [("p", a, np & 1), ("v", st)], [("o", a)])]
                        np += 1
                    issue.append(("mma", [("v_empty", st)], [], []))
            nk += n
        issue.append(wait(("item_full", end & 1), end >> 1))
        roles.append(issue)
    for _ in range(turners):
        turn, nk = [], 0
        for ni in range(end):
            turn += [wait(("item_full", ni & 1), ni >> 1), ("arrive", ("item_empty", ni & 1))]
            for _ in range(tiles[ni]):
                turn += [wait(("raw_full", nk % nraw), nk // nraw), ("write", ("raw", nk % nraw))]      # (reads it: not beside a copy)
                for x in "kv":
                    if nk >= nst:
                        turn.append(wait((x + "_empty", nk % nst), nk // nst - 1))
                    turn += [("write", (x, nk % nst)), ("arrive", (x + "_full", nk % nst))]
                    if x == "k":
                        turn.append(("arrive", ("raw_empty", nk % nraw)))
                nk += 1
        turn.append(wait(("item_full", end & 1), end >> 1))
        roles.append(turn)
    for a in range(2):
        s, ns, nk, joined = [], 0, 0, {}

        def join(bar, meet):
            s.append(("join", (bar,), a))
            if meet:                                             # bar.sync
                s.append(("meet", (bar,), joined.get(bar, 0)))
            joined[bar] = joined.get(bar, 0) + 1
        for ni, nn in enumerate(items):
            s += [wait(("item_full", ni & 1), ni >> 1), ("arrive", ("item_empty", ni & 1)), wait(("q_full",), ni)]
            if nn[a]:
                s.append(("read", ("q",)))
            s.append(("arrive", ("q_empty",)))
            for j in range(nn[a]):
                jt = 2 * j + a if nn[2] else j
                s += [wait(("s_full", a), ns), ("read", ("s", a)), ("arrive", ("s_read", a)), wait(("v_full", (nk + jt) % nst), (nk + jt) // nst)]
                if j:
                    s += [wait(("o_full", a, (ns - 1) & 1), (ns - 1) >> 1, True)]        # only where a row's reference moves
                if ns >= 2:
                    s.append(wait(("o_full", a, ns & 1), (ns - 2) >> 1))
                turn = nn[1] >= 3 and j == 0
                if turn and a:
                    join("bar1", True)
                s.append(("write", ("p", a, ns & 1)))
                if turn and not a:
                    join("bar1", False)
                s.append(("arrive", ("p_full", a, ns & 1)))
                ns += 1
            if nn[a]:
                s += [wait(("o_full", a, (ns - 1) & 1), (ns - 1) >> 1), ("read", ("o", a))]
            if nn[2]:
                join("bar2", True)
                if not a:
                    s.append(("read", ("o", 1)))
                join("bar3", True)
            nk += tiles[ni]
        s.append(wait(("item_full", end & 1), end >> 1))
        roles.append(s)
    return roles


def explore(items, nst=3, nraw=3, turners=1, only=None, drop=None, codes=True):
    """What can go wrong (barrier_explorer).  only: the query tile whose roles are run (the other's arrivals are taken out), which keeps the
    number of states small; so does codes: False, the codes of every tile are always there.  drop: a wait that is left out."""
    roles = programs(items, nst, nraw, turners)
    need = {"item_empty": 4 + turners, "k_empty": 2, "v_empty": 2, "q_empty": 4, "k_full": turners, "v_full": turners, "raw_empty": turners}
    if only is not None:
        roles = [roles[0], roles[1 + only], *roles[3:-2], roles[-2 + only]]
        need |= {"item_empty": 2 + turners, "k_empty": 1, "v_empty": 1, "q_empty": 2}
        roles = [[op for op in r if op[0] == "mma" or op[1][0][:3] != "bar"] for r in roles]
    if not codes:
        roles = [[op for op in r if op[0] == "mma" or op[1][0][:3] != "raw"] for r in roles]
    if drop:
        roles = [[op for op in r if not (op[0] == "wait" and op[1][0] == drop)] for r in roles]
    return barrier_explorer.explore(roles, need)


@pytest.mark.parametrize("items", [[(1, 0)], [(1, 1)], [(1, 2)], [(2, 1, 1)], [(1, 0), (1, 0)]], ids=str)
def test_every_wait_of_a_prompt_ends_in_every_order(items):
    assert not explore(items, 2, 2, codes=False)


@pytest.mark.parametrize("nst", [2, 3])
@pytest.mark.parametrize("items", [[(4, 5)], [(2, 3), (1, 0), (3, 3)], [(1, 1)] * 4, [(4, 5), (2, 0)], [(3, 2, 1), (2, 2)], [(1, 1, 1)] * 3, [(2, 4), (3, 3)]], ids=str)
@pytest.mark.parametrize("only", [0, 1])
def test_every_wait_of_one_query_tile_ends_in_every_order(items, nst, only):
    assert not explore(items, nst, only=only, codes=False)


@pytest.mark.parametrize("items", [[(4, 0)], [(1, 0)] * 3, [(2, 0), (3, 0)]], ids=str)
@pytest.mark.parametrize("nraw,turners", [(2, 1), (3, 1), (2, 2)])
def test_every_wait_for_codes_ends_in_every_order(items, nraw, turners):
    assert not explore(items[:2 if turners == 2 else 3], 2, nraw, turners, only=0)


@pytest.mark.parametrize("drop", ["o_full", "p_full", "s_read", "k_empty", "v_empty", "q_empty", "raw_full", "raw_empty"])
def test_the_exploration_finds_a_missing_wait(drop):
    assert explore([(3, 3), (2, 1)], 2, 2, only=0, drop=drop)


# ------------------------------------------------------------------------------------------------- shares of long contexts

def share_programs(pieces, stages, warps):
    """The producer and the computing warps of a share: pieces of so many stages each."""
    prod, comp, n = [], [], 0
    for p, tiles in enumerate([*pieces, 0]):
        if p >= 2:
            prod.append(wait(("p_empty", p & 1), (p >> 1) - 1))
        comp.append(wait(("p_full", p & 1), p >> 1))
        if p == len(pieces):                                     # the end: t0 == t1
            prod += [("write", ("piece", p & 1)), ("arrive", ("p_full", p & 1))]
            break
        prod += [("write", ("piece", p & 1)), ("load", ("p_full", p & 1), ("q", p & 1))]
        comp += [("write", ("q", p & 1)), ("arrive", ("p_empty", p & 1))]      # (reads it: not beside a copy)
        for _ in range(tiles):
            if n >= stages:
                prod.append(wait(("empty", n % stages), n // stages - 1))
            prod.append(("load", ("full", n % stages), ("ring", n % stages)))
            comp += [wait(("full", n % stages), n // stages), ("write", ("ring", n % stages)), ("arrive", ("empty", n % stages))]
            n += 1
    return [prod] + [comp] * warps


def explore_share(pieces, stages, warps, drop=None):
    roles = share_programs(pieces, stages, warps)
    if drop:
        roles = [[op for op in r if not (op[0] == "wait" and op[1][0] == drop)] for r in roles]
    return barrier_explorer.explore(roles, {"empty": warps, "p_empty": warps})


@pytest.mark.parametrize("pieces", [[1], [5], [1, 1, 1, 1, 1], [2, 7, 1], [4, 4]], ids=str)
@pytest.mark.parametrize("stages,warps", [(3, 2), (4, 2), (3, 4)])
def test_every_wait_of_a_share_ends_in_every_order(pieces, stages, warps):
    assert not explore_share(pieces, stages, warps)


@pytest.mark.parametrize("drop", ["full", "empty", "p_full", "p_empty"])
def test_the_exploration_finds_a_missing_wait_of_a_share(drop):
    assert explore_share([2, 3, 1, 2], 3, 2, drop)
