"""The barriers of the tcgen05 tree attention, searched exhaustively in a small model (CPU suite).

A parity wait tells the waiter only whether the barrier's current phase has the other parity.  It is the wait that was
meant only if the phase before is complete and the phase after is not, so every pair of roles that share a barrier
needs an order between them.  The model has the roles of ``attn_tree_tc.cu`` as straight-line programs over
barriers: K and V loads that complete in any order (8 bits: conversions, in order), the issuing thread and the
softmax of both streams; all interleavings are tried.  Faults: a product that reads a stage which does not
hold its tile, and a state in which nobody can go on.  The numbers come from the kernel's source.
"""

import re
from collections import deque
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "thesis_b200" / "csrc" / "attn_tree_tc.cu").read_text()


def stages(q8):
    eight, sixteen = re.search(r"int NS = Q8 \? (\d+) : (\d+);", SOURCE).groups()
    return int(eight if q8 else sixteen)


def programs(pieces, NS, q8, weights_first, ml_issuer):
    """Roles and barriers.  ``pieces``: (key tiles, whether it has more than one row tile).  Ops: ("w", barrier, phase),
    ("a", barrier), ("load", "k" | "v", tile), ("read", "k" | "v", tile)."""
    n_pieces = len(pieces)
    first = [sum(n for n, _ in pieces[:i]) for i in range(n_pieces)]
    count = {("ml",): 2 + ml_issuer}
    for s in range(NS):
        count.update({("kfull", s): 1, ("vfull", s): 1, ("kempty", s): 2, ("vempty", s): 2})
    for x in (0, 1):
        count.update({("s_full", x): 1, ("s_free", x): 1, ("p_ready", x): 1, ("pv_done", x): 1})
    count.update({("q_ready",): 2, ("o_done",): 2, ("epi",): 2})
    prog = {"K": [], "V": []} if q8 else {"K": []}                      # over 16 bits one thread asks for K and V in turn
    for c in range(sum(n for n, _ in pieces)):
        for role, kind in (("K", "k"), ("V" if q8 else "K", "v")):
            if c >= NS:
                prog[role].append(("w", (kind + "empty", c % NS), c // NS - 1))
            prog[role].append(("load", kind, c))
    for x in (0, 1):
        mma, soft, n_q, n_p, n_s, n_ml = [], [], 0, 0, 0, 0
        for p, (nt, two) in enumerate(pieces):
            step, t0 = (1, 0) if two else (2, x)
            free = 1 if two else 2
            mma.append(("w", ("q_ready",), p))
            if ml_issuer and x == 1 and not two:
                mma.append(("a", ("ml",)))
            for i in range(t0 - step, nt, step):
                if i + step < nt:
                    c = first[p] + i + step
                    if n_q:
                        mma.append(("w", ("s_free", x), n_q - 1))
                    n_q += 1
                    mma += [("w", ("kfull", c % NS), c // NS), ("read", "k", c), ("a", ("s_full", x))] + [("a", ("kempty", c % NS))] * free
                if i >= 0:
                    c = first[p] + i
                    waits = [("w", ("vfull", c % NS), c // NS), ("w", ("p_ready", x), n_p)]
                    n_p += 1
                    mma += waits[::-1] if weights_first and i == t0 else waits
                    mma += [("read", "v", c), ("a", ("pv_done", x))] + [("a", ("vempty", c % NS))] * free
            mma.append(("a", ("o_done",)))
        for p in range(-1, n_pieces):                                   # a turn: the next Q out, the last output, the next tiles
            if p >= 0 and not pieces[p][1]:
                soft += [("a", ("ml",)), ("w", ("ml",), n_ml)]
                n_ml += 1
            if p + 1 < n_pieces:
                soft.append(("a", ("q_ready",)))
            if p >= 0:
                soft += [("w", ("o_done",), p), ("a", ("epi",))]
            if p + 1 < n_pieces:
                nt, two = pieces[p + 1]
                start = 0 if two else x
                for i in range(start, nt, 1 if two else 2):
                    soft += [("w", ("s_full", x), n_s), ("a", ("s_free", x))]
                    if n_s:
                        soft.append(("w", ("pv_done", x), n_s - 1))
                    if i == start and p >= 0:
                        soft.append(("w", ("epi",), p))
                    soft.append(("a", ("p_ready", x)))
                    n_s += 1
        prog["M%d" % x], prog["S%d" % x] = mma, soft
    return prog, count


def fault(pieces, NS, q8, weights_first, ml_issuer):
    """The first fault that some interleaving has, or None."""
    prog, count = programs(pieces, NS, q8, weights_first, ml_issuer)
    roles, bars = list(prog), list(count)
    at = {b: i for i, b in enumerate(bars)}

    def arrive(bs, b):
        i = at[b]
        done, left = bs[i]
        done, left = (done + 1, count[b]) if left == 1 else (done, left - 1)
        return bs[:i] + ((done, left),) + bs[i + 1:]

    start = ((0,) * len(roles), tuple((0, count[b]) for b in bars), frozenset(), (-1,) * NS, (-1,) * NS)
    seen, todo = {start}, deque([start])
    while todo:
        pcs, bs, flying, kt, vt = todo.popleft()
        after = []
        for a, role in enumerate(roles):
            if pcs[a] == len(prog[role]):
                continue
            op = prog[role][pcs[a]]
            nxt = pcs[:a] + (pcs[a] + 1,) + pcs[a + 1:]
            if op[0] == "w":
                if bs[at[op[1]]][0] % 2 != op[2] % 2:                   # the current phase has the other parity
                    after.append((nxt, bs, flying, kt, vt))
            elif op[0] == "a":
                after.append((nxt, arrive(bs, op[1]), flying, kt, vt))
            elif op[0] == "load":
                if not (q8 and any(k == op[1] for k, _ in flying)):
                    after.append((nxt, bs, flying | {op[1:]}, kt, vt))
            else:
                holds = (kt if op[1] == "k" else vt)[op[2] % NS]
                if holds != op[2]:
                    return "%s reads tile %d of %s, the stage holds %d" % (role, op[2], op[1], holds)
                after.append((nxt, bs, flying, kt, vt))
        for kind, c in flying:
            if kind == "v" and any(k == "v" and o < c for k, o in flying):
                continue                                                # V tiles are checked or converted in order
            s, left, full = c % NS, flying - {(kind, c)}, arrive(bs, (kind + "full", c % NS))
            if kind == "k":
                after.append((pcs, full, left, kt[:s] + (c,) + kt[s + 1:], vt))
            else:
                after.append((pcs, full, left, kt, vt[:s] + (c,) + vt[s + 1:]))
        if not after and any(pcs[a] < len(prog[r]) for a, r in enumerate(roles)):
            return "nobody can go on: " + ", ".join("%s at %s" % (r, prog[r][pcs[a]][:2]) for a, r in enumerate(roles) if pcs[a] < len(prog[r]))
        for n in after:
            if n not in seen:
                seen.add(n)
                todo.append(n)
    return None


# every V wait ordered and every arrival there: what is left is the ring itself
@pytest.mark.parametrize("pieces", [[(6, False)], [(3, False), (2, False)], [(1, False), (3, False)], [(2, True), (3, False)]], ids=str)
def test_k_stages_hold_the_tile_that_a_product_reads(pieces):
    assert fault(pieces, stages(False), False, True, 1) is None


def first_weights_before_v():
    return re.search(r"if \(i == t0 && !\(ok = mbar_wait\(smem_u32\(&ct\.p_ready", SOURCE) is not None


# The two stages of the 8-bit tiles change hands between pieces: after an odd one a stream's first V stage was the other's.
@pytest.mark.parametrize("pieces", [[(3, False), (3, False)], [(1, False), (2, False), (2, False)], [(3, False), (2, True)]], ids=str)
def test_first_v_of_a_piece_is_waited_for_in_its_own_phase(pieces):
    assert fault(pieces, stages(True), True, first_weights_before_v(), 1) is None


def issuer_arrivals_on_ml():
    """How many arrivals beside the eight softmax warps' complete ml_ready."""
    return int(re.search(r"mbar_init\(smem_u32\(&ct\.ml_ready\), (\d+)\)", SOURCE).group(1)) - 8


# A piece of one key tile leaves stream 1 without a product: its issuing thread must not fall a phase of q_ready behind.
@pytest.mark.parametrize("pieces", [[(1, False)] * 3, [(1, False), (1, True), (1, False)], [(2, False), (1, False), (1, False)]], ids=str)
def test_pieces_of_one_tile_do_not_run_ahead_of_stream_1(pieces):
    assert fault(pieces, stages(True), True, first_weights_before_v(), issuer_arrivals_on_ml()) is None
