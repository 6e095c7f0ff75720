"""The waits of prompt attention (csrc/attn_prompt.cu) in a model on the CPU: every order in which copies land, products end and warps go on (no GPU needed).

A barrier's wait gets a bit and passes where the last phase that is over has it: it tells a phase from its neighbours alone. So each wait stands behind something that keeps the barrier within one phase of the one that is
meant. The model has the kernel's threads as lists of waits, copies, commits and arrivals, and goes through all states that they can reach: no wait may pass before its phase is over, and all threads come to their end."""
import pytest


def threads(tiles, stages, parts, *, take_waits=True, one_pv=False):
    """-> names of the threads' steps: (wait, barrier, phase), (may, barrier, phase) which is asked or left out, (copy, barrier), (commit, barrier), (arrive, barrier). parts: of a tile's V, a weights' warp for each."""
    pv = (lambda n: (("pv", 0), n)) if one_pv else (lambda n: (("pv", n & 1), n >> 1))
    full = lambda kind, n, p=0: ((kind, n % stages, p), n // stages)  # noqa: E731
    k_copies, v_copies, scores, outputs = [], [], [], []
    for n in range(tiles):
        if stages == 1:   # a warp of its own fetches what is free, K and V in any order
            if n:
                k_copies.append(("wait", *full("k_empty", n - 1)))
            k_copies.append(("copy", full("k_full", n)[0]))
            for p in range(parts):
                if n:
                    v_copies.append(("wait", *full("v_empty", n - 1, p)))
                v_copies.append(("copy", full("v_full", n, p)[0]))
        else:             # the products' warps fetch: two tiles ahead, then each again as soon as its products are through
            for mine, name in ((scores, "k"), (outputs, "v")):
                if n == 0:
                    mine.extend(("copy", full(name + "_full", i)[0]) for i in range(min(stages, tiles)))
                elif n + 1 < tiles:
                    mine.append(("wait", *full(name + "_empty", n - 1)))
                    mine.append(("copy", full(name + "_full", n + 1)[0]))
        if n >= 2:
            scores.append(("wait", *pv(n - 2)))
        scores += [("wait", *full("k_full", n)), ("commit", full("k_empty", n)[0]), ("commit", ("s", n & 1))]
        for p in range(parts):
            outputs.append(("wait", *full("v_full", n, p)))
            for h in range(2 // parts):
                outputs.append(("wait", ("w", n & 1, p + h), n >> 1))
            outputs.append(("commit", full("v_empty", n, p)[0]))
        outputs.append(("commit", pv(n)[0]))
    weights = []
    hides = lambda n: n >= tiles - stages  # noqa: E731   tiles of the block's own rows
    for warp in range(2):
        mine, part = [], warp % parts
        for n in range(tiles):
            if n == 0 and hides(0):
                mine.append(("wait", *full("v_full", 0, part)))
            mine.append(("wait", ("s", n & 1), n >> 1))
            if n:
                mine.append(("may", *pv(n - 1)))   # where a reference moves
            if n and hides(n):
                if stages == 1 and take_waits:
                    mine.append(("wait", *pv(n - 1)))
                mine.append(("wait", *full("v_full", n, part)))
            mine += [("arrive", ("w", n & 1, 0)), ("arrive", ("w", n & 1, 1))]
        mine.append(("wait", *pv(tiles - 1)))
        weights.append(mine)
    return [k_copies, v_copies, scores, outputs, *weights]


def explore(programs):
    """-> the first wait that passes early, or "stuck", or None after all states."""
    bars = sorted({s[1] for p in programs for s in p}, key=repr)
    number = {b: i for i, b in enumerate(bars)}
    code = [[(s[0], number[s[1]], s[2] if len(s) > 2 else 0) for s in p] for p in programs]
    need = [2 if b[0] == "w" else 1 for b in bars]
    start = (tuple(0 for _ in code), tuple(0 for _ in bars), frozenset(), tuple(() for _ in code))   # places, arrivals, copies on their way, commits on their way
    seen, todo = {start}, [start]
    while todo:
        at, came, flying, queues = todo.pop()
        nexts = []
        arrive = lambda b: came[:b] + (came[b] + 1,) + came[b + 1:]  # noqa: E731
        for b in flying:
            nexts.append((at, arrive(b), flying - {b}, queues))
        for t, q in enumerate(queues):
            if q:   # products of a thread end in order
                nexts.append((at, arrive(q[0]), flying, queues[:t] + (q[1:],) + queues[t + 1:]))
        for t, p in enumerate(code):
            if at[t] == len(p):
                continue
            what, b, phase = p[at[t]]
            on = at[:t] + (at[t] + 1,) + at[t + 1:]
            if what in ("wait", "may"):
                over = came[b] // need[b]
                if (over & 1) != (phase & 1):
                    if over <= phase:
                        return t, what, bars[b], phase, over
                    nexts.append((on, came, flying, queues))
                if what == "may":
                    nexts.append((on, came, flying, queues))
            elif what == "copy":
                assert b not in flying
                nexts.append((on, came, flying | {b}, queues))
            elif what == "commit":
                nexts.append((on, came, flying, queues[:t] + (queues[t] + (b,),) + queues[t + 1:]))
            else:
                nexts.append((on, arrive(b), flying, queues))
        if not nexts and any(a < len(p) for a, p in zip(at, code)):
            return "stuck"
        for s in nexts:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return None


@pytest.mark.parametrize("stages,parts", [(1, 2), (2, 1)])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4])
def test_no_wait_passes_early(stages, parts, tiles):
    assert explore(threads(tiles, stages, parts)) is None


def test_the_model_finds_waits_that_pass_early():
    """One stage: values of the last tile looked at without a wait for the products of the tile before; and one barrier for the products of all tiles."""
    for tiles in (2, 3):
        found = explore(threads(tiles, 1, 2, take_waits=False))
        assert found[1:3] == ("wait", ("v_full", 0, found[2][2])) and found[3] == tiles - 1 and found[4] == tiles - 2, found
    assert explore(threads(2, 2, 1, take_waits=False)) is None   # two stages: the scores of a tile are formed behind the products of the last but one
    assert explore(threads(4, 2, 1, one_pv=True)) is not None
