"""CPU: the hand-overs in the forward kernels of differential attention (``ops/csrc/attn_diff_fwd.cu``), of the scaled
queries and of the rows' reference, by walking every order in which their events can happen.

The softmax warps multiply the queries of a walk (one map over a segment's K/V tiles) by the scale in shared
memory, each a share of them; the issuing thread makes scores when all shares are there.  Which barrier and which
phase stand for a walk is read from the kernel's source.  Modelled as the hardware has them: a barrier counts
arrivals, whoever makes them, and a wait sees the parity of the phase only."""
import itertools
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


# ---- O and its reference: what both kernels' groups of softmax warps, the issuer and the tensor core do to one another ----
KERNELS = {"primal": ("-- primal ---", "-- tangent ---"), "tangent": ("-- tangent ---", "-- merge ---")}
STEP = {"own": r"mbar_wait\(&s\.o_done(\[t\])?\[g\], par \^ 1", "scores": r"mbar_wait\(&s\.s_full(\[t\])?\[g\], par,",
        "see": r"ref_of_step\(", "publish": r"publish_ref\(",
        "other": r"mbar_wait\(&s\.o_done(\[t\])?\[g \^ 1\], g == 0 \? par \^ 1 : par", "rescale": r"tmem_st\d+\(tb \+ [PT]_COL_O",
        "P": r"mbar_arrive\(&s\.p_full(\[t\])?\[g\]\)"}


def step_events(kernel):
    """The order of a step's events in the source (``own``, if it is there)."""
    text = open(SOURCE).read()
    a, b = (text.index(x) for x in KERNELS[kernel])
    text = text[a:b]
    body = text[text.index("for (int j = j_own"):text.index("// ---- epilogue of this")]
    at = {}
    for name, pattern in STEP.items():
        hits = [m.start() for m in re.finditer(pattern, body)]
        assert len(hits) == 1 or (name == "own" and not hits), (kernel, name, len(hits))
        if hits:
            at[name] = hits[0]
    return sorted(at, key=at.get)


def rescale_orders(order, kernel, segments, outgrown):
    """None, or what goes wrong in some order of events: a warp stands for a group, ``outgrown`` are the steps that move
    the reference.  Products run in the order in which they are issued; the arrival that a commit stands for comes any
    time after them, in order on one barrier and in none between two; a wait sees the parity of the phase only."""
    per = 2 if kernel == "tangent" else 1
    walks = [n for n in segments for _ in range(per)]
    first = [sum(walks[:w]) for w in range(len(walks) + 1)]
    warps = []
    for g in (0, 1):
        ev = []
        for w, n_j in enumerate(walks):
            for n in range(first[w], first[w] + n_j):
                if n % 2 == g:
                    moves = n in outgrown and n != first[w]
                    ev += [(e, n) for e in order if moves or e not in ("other", "rescale")]
            ev += [("final", w), ("sums", w), ("summed", w), ("read", w)]
        warps.append(ev)
    issuer = []
    for w, n_j in enumerate(walks):
        make = lambda n: [("run", "S", n), ("commit", f"s{n % 2}")]
        if per == 2 and w:                  # the next walk's queries are scaled behind the last of this one's steps
            issuer.append(("steps", w - 1))
        for n in range(first[w], first[w] + min(n_j, 2)):
            issuer += make(n)
        if w:
            issuer.append(("read", w - 1))
        for n in range(first[w], first[w] + n_j):
            issuer += [("P", n), ("run", "O", n), ("commit", f"o{n % 2}")]
            if n + 1 == first[w + 1]:
                issuer.append(("commit", "final"))
            if n + 2 < first[w + 1]:
                issuer += make(n + 2)
    queue = [e for e in issuer if e[0] in ("run", "commit")]
    issued = [sum(e[0] in ("run", "commit") for e in issuer[:i]) for i in range(len(issuer) + 1)]
    runs = [i for i, e in enumerate(queue) if e[0] == "run"]
    bars = sorted({e[1] for e in queue if e[0] == "commit"})
    commits = [[i for i, e in enumerate(queue) if e == ("commit", b)] for b in bars]
    where = [{e: i for i, e in enumerate(ev)} for ev in warps]
    behind = lambda pos, e: all(e not in where[g] or pos[g] > where[g][e] for g in (0, 1))
    last = [[max([where[g][("P", n)] for n in range(first[w], first[w + 1]) if n % 2 == g], default=-1)
             for w in range(len(walks))] for g in (0, 1)]
    products = [sum(queue[i][1] == "O" for i in runs[:r]) for r in range(len(runs) + 1)]
    start = ((0, 0), 0, 0, (0,) * len(bars))
    seen, todo = {start}, [start]
    while todo:
        pos, ip, ran, arrived = state = todo.pop()
        passes = lambda b, parity: (arrived[bars.index(b)] & 1) != parity
        nxt = []
        if ip < len(issuer):
            kind, n = issuer[ip][0], issuer[ip][-1]
            ok = True
            if kind == "P":
                ok = behind(pos, ("P", n))
            elif kind == "read":
                ok = behind(pos, ("read", n))
            elif kind == "steps":
                ok = all(pos[g] > last[g][n] for g in (0, 1))
            if ok:
                nxt.append((pos, ip + 1, ran, arrived))
        if ran < len(runs) and runs[ran] < issued[ip]:
            nxt.append((pos, ip, ran + 1, arrived))
        over = min(issued[ip], runs[ran] if ran < len(runs) else len(queue))
        for b in range(len(bars)):
            if arrived[b] < len(commits[b]) and commits[b][arrived[b]] < over:
                nxt.append((pos, ip, ran, tuple(a + (i == b) for i, a in enumerate(arrived))))
        for g in (0, 1):
            if pos[g] == len(warps[g]):
                continue
            kind, n = warps[g][pos[g]]
            k = n // 2 & 1                   # phase of the step in its group
            ok = True
            if kind == "own":
                ok = passes(f"o{g}", k ^ 1)
            elif kind == "scores":
                ok = passes(f"s{g}", k)
            elif kind == "see":
                ok = n == 0 or behind(pos, ("publish", n - 1))
            elif kind == "other":
                ok = passes(f"o{g ^ 1}", k ^ 1 if g == 0 else k)
            elif kind == "rescale" and products[ran] != n:
                return f"O is moved to the reference of step {n} with {products[ran]} products run"
            elif kind == "final":
                ok = passes("final", n & 1)
            elif kind == "summed":
                ok = behind(pos, ("sums", n))
            elif kind == "read" and products[ran] != first[n + 1]:
                return f"the result of walk {n} is read with {products[ran]} products run"
            if ok:
                nxt.append((tuple(p + (i == g) for i, p in enumerate(pos)), ip, ran, arrived))
        if not nxt and (ip < len(issuer) or any(pos[g] < len(warps[g]) for g in (0, 1))):
            return f"no event can happen any more: {state}"
        for s in nxt:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return None


@pytest.mark.parametrize("kernel,segments", [("primal", (2,)), ("primal", (5,)), ("primal", (2, 3)), ("primal", (1, 4)),
                                             ("tangent", (1,)), ("tangent", (2,)), ("tangent", (3,)), ("tangent", (1, 2))])
def test_o_is_only_moved_between_its_products(kernel, segments):
    order = step_events(kernel)
    steps = sum(segments) * (2 if kernel == "tangent" else 1)
    for some in itertools.product((False, True), repeat=steps - 1):
        outgrown = {n + 1 for n, x in enumerate(some) if x}
        wrong = rescale_orders(order, kernel, segments, outgrown)
        assert wrong is None, (outgrown, wrong)
