"""The operators for several continuations of a sequence, from their definitions
in include/q4rdna.h: whole numbers in Python, sums in 64 bits."""
import numpy as np

BLOCK = 64


def tree(past, counts, parents):
    """(positions, seen) of the step's tokens; seen as unsigned."""
    positions, seen, at = [], [], 0
    for p, c in zip(past, counts):
        mine = []
        for j in range(c):
            up = parents[at + j]
            if not -1 <= up < j or (up >= 0 and mine[up] == 0):
                mine.append(0)
            else:
                mine.append(1 << j | (mine[up] if up >= 0 else 0))
        positions += [p + bin(s).count("1") - 1 if s else -1 for s in mine]
        seen += mine
        at += c
    return positions, seen


def visible(past, count, seen, window):
    """[count, past + count] truth values: what each drafted token of one
    sequence sees of the cached tokens and then of the drafted ones."""
    seen = [int(s) & ((1 << count) - 1) for s in seen]
    stands = [past - 1 + bin(s).count("1") for s in seen]
    out = np.zeros((count, past + count), dtype=bool)
    for j in range(count):
        out[j, :past] = True
        out[j, past:] = [seen[j] >> a & 1 for a in range(count)]
        if window:
            out[j, :past] &= np.arange(past) > stands[j] - window
            out[j, past:] &= np.array(stands) > stands[j] - window
    return out


def attend(q, keys, values, sees, scale):
    """q [rows, dim] over keys and values [tokens, dim], sees [rows, tokens]:
    (out, lse).  Tokens that a row does not see count for nothing, whatever is
    in them; a row that sees nothing is zero."""
    out, lse = np.zeros(q.shape), np.full(q.shape[0], -np.inf)
    for r in range(q.shape[0]):
        k, v = keys[sees[r]], values[sees[r]]
        if len(k):
            s = scale * (k @ q[r])
            e = np.exp(s - s.max())
            out[r] = e @ v / e.sum()
            lse[r] = s.max() + np.log(e.sum())
    return out, lse


def beam_select(logits, scores, count):
    """(scores, rows, tokens), logits [groups, beams, vocab] in 64 bits."""
    groups, beams, vocab = logits.shape
    logits = logits.copy()
    total = np.full(logits.shape, -np.inf)
    for g in range(groups):
        for b in range(beams):
            x, s = logits[g, b], 0.0 if scores is None else float(scores[g, b])
            if np.isfinite(s) and not np.isnan(x).any() and np.isfinite(x.max()):
                total[g, b] = s + (x - (x.max() + np.log(np.exp(x - x.max()).sum())))
            else:
                logits[g, b] = -np.inf
    flat = total.reshape(groups, -1)
    # by total, row, logit, token
    order = np.stack([np.lexsort((np.arange(beams * vocab), -logits[g].reshape(-1), np.arange(beams * vocab) // vocab, -flat[g]))
                      for g in range(groups)])[:, :count]
    return np.take_along_axis(flat, order, 1), order // vocab + np.arange(groups)[:, None] * beams, order % vocab


def fork(past, table, slots, parents, pages, room, slot_count, kept=()):
    """(past, table, slots, copies, faults): copies are (from, to, block) of the
    slots' open blocks."""
    n, width, faults = len(past), len(table[0]), 0
    up = []
    for p in parents:
        bad = p != -1 and not (0 <= p < n and 0 <= past[p] <= BLOCK * width and 0 <= slots[p] < slot_count)
        faults += bad
        up.append(-1 if bad else p)
    vacant = [slots[q] for q in range(n) if q not in up]
    new_past, new_slots, copies = [], [], []
    for i in range(n):
        first = up[i] >= 0 and up[i] not in up[:i]
        slot = slots[up[i]] if first else vacant.pop(0)
        if not first and up[i] >= 0:
            if not 0 <= slot < slot_count:
                faults += 1
                up[i] = -1
            else:
                m = past[up[i]]
                copies += [(slots[up[i]], slot, b) for b in (m // BLOCK, m // BLOCK - 1) if 0 <= b and b * BLOCK < m]
        new_slots.append(slot)
        new_past.append(past[up[i]] if up[i] >= 0 else 0)
    rows = [list(table[u][:m // BLOCK]) if u >= 0 else [] for u, m in zip(up, new_past)]
    held = {p for row in rows for p in row} | {p for p in range(pages) if p in kept}
    free = [p for p in range(pages) if p not in held]
    for u, m, row in zip(up, new_past, rows):
        end = min(width, -(-(m + room) // BLOCK)) if u >= 0 else 0
        while len(row) < end:
            faults += not free
            row.append(free.pop(0) if free else -1)
        row += [-1] * (width - len(row))
    return new_past, rows, new_slots, copies, faults
