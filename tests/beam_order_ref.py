"""The reordering of beams' block tables by plain loops over Python integers."""


def reorder(tables, parents, contexts, free, start, block):
    """tables: rows of every beam; parents: for each request; contexts: a count for each request.
    Returns (tables, copied_from, free list, first free entry, lacking, unlisted, copies), with
    copies [(from, to, tokens)]."""
    beams, width = len(parents[0]), len(tables[0])
    new, copied, copies, lacking, released = [list(t) for t in tables], [], [], 0, []
    for r, (chosen, context) in enumerate(zip(parents, contexts)):
        old = tables[r * beams:(r + 1) * beams]
        context = max(context, 0)
        full, rest = context // block, context % block
        known = [0 <= p < beams for p in chosen]
        lacking += known.count(False)
        kept = {p for p, ok in zip(chosen, known) if ok}
        moved = [-1] * beams
        for c in range(min(width, full + (1 if rest else 0))):
            column = [old[b][c] for b in range(beams)]
            held = {column[p] for p in kept}
            left = []
            for b in range(beams):
                if column[b] >= 0 and column[b] not in held and column[b] not in left:
                    left.append(column[b])
            taken = set()
            for j, p in enumerate(chosen):
                to = column[p] if known[j] else -1
                if c == full and known[j]:
                    if to >= 0 and to in taken:
                        source, to = to, left.pop(0) if left else -1
                        if to >= 0:
                            moved[j] = source
                            copies.append((source, to, rest))
                    elif to >= 0:
                        taken.add(to)
                    if to < 0:
                        lacking += 1
                new[r * beams + j][c] = to
            released += left
        copied += moved
    start = min(max(start, 0), len(free))
    free = list(free)
    room = released[max(len(released) - start, 0):]
    free[start - len(room):start] = room
    return new, copied, free, start - len(room), lacking, len(released) - len(room), copies
