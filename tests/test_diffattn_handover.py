"""CPU: the hand-over of the scaled queries in the tangent kernel of differential attention
(``ops/csrc/attn_diff_fwd.cu``), by walking every order in which its events can happen.

The softmax warps multiply the queries of a walk (one map over a segment's K/V tiles) by the scale in shared
memory, each a share of them; the issuing thread makes scores when all shares are there.  Which barrier and which
phase stand for a walk is read from the kernel's source.  Modelled as the hardware has them: a barrier counts
arrivals, whoever makes them, and a wait sees the parity of the phase only."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "imfvideo_b200", "ops",
                      "csrc", "attn_diff_fwd.cu")
WARPS = 4                                 # two of either group stand for the four


def barriers():
    """(walk -> barrier of the arrivals, walk -> (barrier, parity) of the issuer's wait)."""
    text = open(SOURCE).read()
    index = r"&s\.q_ready(?:\[([^\]]*)\])?"
    (arrive,) = re.findall(r"mbar_arrive\(" + index + r"\)", text)
    ((bar, parity),) = re.findall(r"mbar_wait\(" + index + r", ([^?:]*?), abort_flag", text)
    number = lambda e: eval(re.sub(r"\(uint32_t\)", "", e or "0"), {}, names)

    def at(expr, w):
        names.update(w=w, walk=w, qs=w & 1)
        return number(expr)
    names = {}
    return (lambda w: at(arrive, w)), (lambda w: (at(bar, w), at(parity, w)))


def program(segments):
    """What each warp and the issuer do, in order; ``segments``: K/V tiles of each, two walks a segment."""
    walks = [n for n in segments for _ in range(2)]
    first = [sum(walks[:w]) for w in range(len(walks) + 1)]
    warps = []
    for i in range(WARPS):
        ev = [("scale", 0)]
        for w, n_j in enumerate(walks):
            for n in range(first[w], first[w] + n_j):
                if n % 2 == i // (WARPS // 2):
                    ev += [("scores", n), ("P", n)]
            if w + 1 < len(walks):
                ev.append(("scale", w + 1))
            ev += [("o_final", w), ("sums", w), ("summed", w), ("free", w)]
        warps.append(tuple(ev))
    issuer = []
    for w, n_j in enumerate(walks):
        issuer += [("ready", w)] + [("make", first[w] + j) for j in range(min(n_j, 2))]
        if w:
            issuer.append(("freed", w - 1))
        for j in range(n_j):
            issuer.append(("product", first[w] + j))
            if j + 2 < n_j:
                issuer.append(("make", first[w] + j + 2))
        issuer.append(("final", w))
    return warps, tuple(issuer)


def walk_orders(segments):
    """None, or what goes wrong in some order of events."""
    arrive, wait = barriers()
    warps, issuer = program(segments)
    where = [{e: k for k, e in enumerate(ev)} for ev in (*warps, issuer)]
    did = lambda pos, i, e: pos[i] > where[i][e]
    has = lambda i, e: e in where[i]
    everyone = range(WARPS)
    seen, todo = {(0,) * (WARPS + 1)}, [(0,) * (WARPS + 1)]
    while todo:
        pos = todo.pop()
        moved = False
        for i in range(WARPS + 1):
            ev = warps[i] if i < WARPS else issuer
            if pos[i] == len(ev):
                continue
            kind, n = ev[pos[i]]
            if kind == "ready":
                bar, parity = wait(n)
                arrivals = sum(e[0] == "scale" and arrive(e[1]) == bar for j in everyone for e in warps[j][:pos[j]])
                if (arrivals // WARPS & 1) == parity:
                    continue
                late = [j for j in everyone if not did(pos, j, ("scale", n))]
                if late:
                    return f"scores of walk {n} are made while warps {late} have not scaled their share of its queries"
            elif kind == "scale" and n >= 2:     # the queries arrive when the scores of the walk before the last one are made
                if not did(pos, WARPS, ("final", n - 2)):
                    continue
            elif kind == "scores" and not did(pos, WARPS, ("make", n)):
                continue
            elif kind == "product" and not all(did(pos, j, ("P", n)) for j in everyone if has(j, ("P", n))):
                continue
            elif kind == "o_final" and not did(pos, WARPS, ("final", n)):
                continue
            elif kind == "summed" and not all(did(pos, j, ("sums", n)) for j in everyone):
                continue
            elif kind == "freed" and not all(did(pos, j, ("free", n)) for j in everyone):
                continue
            moved = True
            nxt = pos[:i] + (pos[i] + 1,) + pos[i + 1:]
            if nxt not in seen:
                seen.add(nxt)
                todo.append(nxt)
        if not moved and pos != (*map(len, warps), len(issuer)):
            return f"no event can happen any more: {pos}"
    return None


@pytest.mark.parametrize("segments", [(1,), (1, 1), (1, 2), (2,), (2, 1), (3, 1), (1, 3, 1)])
def test_scores_are_made_from_scaled_queries(segments):
    assert walk_orders(segments) is None
