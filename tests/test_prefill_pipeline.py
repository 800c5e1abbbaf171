"""CPU model of the tile kernel's roles (k_attn_prefill): how far ahead of a softmax the group that widens K may run.

The roles meet only in barriers, and a role that goes on never takes a step away from another.  So the furthest that K
gets before a softmax has read what belongs to tile X is where it stands when that softmax stops in front of X and
everything else runs until it cannot.  What K leaves for the softmax beside the operands (the tokens whose page is bad)
lies in a ring, which needs a place for every tile of that lead.
"""
import os
import re

import pytest

SRC = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "q36_b200", "csrc", "kv_prefill.cu")).read()


def ring():
    places = re.search(r"\bbad_s\[(\w+)\]\[2\]", SRC).group(1)
    if not places.isdigit():
        places = re.search(r"constexpr int %s = (\d+)" % places, SRC).group(1)
    return int(places)


def furthest_k(segs, stages, nq, who, stop):
    """segs: (tiles, row tiles that have rows) per span.  K tiles written before softmax `who` has read its tile `stop`."""
    tiles = [(si, j, act, j == n - 1) for si, (n, act) in enumerate(segs) for j in range(n)]
    done = {}
    at = lambda *key: done.get(key, 0)  # noqa: E731

    def bump(*key):
        done[key] = done.get(key, 0) + 1

    def widen(x):
        for y in range(len(tiles)):
            while y >= stages and any(at(x + "_empty", i) <= y - stages for i in range(nq)):
                yield
            bump(x + "_full")

    def issue_s(i):
        n = 0
        for y, (si, j, act, _) in enumerate(tiles):
            if act > i and j == 0:
                want = sum(a > i for _, a in segs[:si + 1])
                while at("q_full", i) < want:
                    yield
            while at("k_full") <= y:
                yield
            if act > i:
                while n >= 2 and at("o_done", i) <= n - 2:
                    yield
                bump("s_full", i)
                n += 1
            bump("k_empty", i)

    def issue_pv(i):
        n = 0
        for y, (_, _, act, last) in enumerate(tiles):
            while at("v_full") <= y:
                yield
            if act > i:
                while at("p_full", i) <= n:
                    yield
                bump("o_done", i)
                n += 1
                if last:
                    bump("o_last", i)
            bump("v_empty", i)

    def softmax(i):
        n = pieces = 0
        for y, (_, j, act, last) in enumerate(tiles):
            if act <= i:
                continue
            if j == 0:
                bump("q_full", i)
            while at("s_full", i) <= n:
                yield
            while i == who and y == stop:
                yield
            bump("p_full", i)
            n += 1
            if last:
                pieces += 1
                while at("o_last", i) < pieces:
                    yield

    roles = [widen("k"), widen("v")] + [r(i) for i in range(nq) for r in (issue_s, issue_pv, softmax)]
    live = list(roles)
    while live:
        before = dict(done)
        for r in list(live):
            try:
                next(r)
            except StopIteration:
                live.remove(r)
        if before == done:
            break
    return at("k_full") - 1, live


# spans of one CTA: both row tiles, then spans whose second row tile is empty, and the other way round
SPANS = {"full": [(40, 2)], "half": [(40, 1)], "full_half": [(12, 2), (40, 1)], "short_half": [(3, 2), (1, 1), (2, 1), (40, 1)],
         "half_full": [(9, 1), (40, 2)], "alternating": [(5, 2), (3, 1)] * 6, "ones": [(1, 2), (1, 1), (1, 1)] * 15}


@pytest.mark.parametrize("name", SPANS)
@pytest.mark.parametrize("stages,nq", [(4, 2), (2, 1)])
def test_bad_pages_of_a_tile_outlast_its_softmax(name, stages, nq):
    assert re.search(r"NQ = DH == 256 \? 1 : 2, R = 128 \* NQ, KT = 64, STAGES = DH == 256 \? 2 : 4;", SRC)      # what is modelled
    segs = [(n, min(a, nq)) for n, a in SPANS[name]]
    total, lead = sum(n for n, _ in segs), 0
    assert furthest_k(segs, stages, nq, -1, -1) == (total - 1, [])                                     # nobody stops: all of it runs through
    for who in range(nq):
        y = 0
        for n, act in segs:
            for stop in range(y, y + n):
                if act > who:
                    lead = max(lead, furthest_k(segs, stages, nq, who, stop)[0] - stop)
            y += n
    print(name, stages, nq, "lead", lead)
    assert lead < ring()
