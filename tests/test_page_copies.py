"""The page manager's copies gathered over several calls, as a scheduler's step gathers them: whatever the
calls between two readings of the table were, the pairs they returned may run in any order or all at
once (no page is one pair's destination and in another pair), and every sequence keeps its tokens."""
import random

import pytest


def independent(pairs):
    src, dst = {s for s, _ in pairs}, [d for _, d in pairs]
    return len(set(dst)) == len(dst) and not src & set(dst)


def shared_tail(irx, pages=8, size=4, tokens=6):
    """Two sequences that share `tokens` tokens, the last page half full."""
    m = irx.Pages(pages, size, 4, 4)
    a = m.open()
    assert m.extend(a, tokens) is None
    b = m.fork(a)
    m.table
    return m, a, b


def test_a_page_freed_after_its_copy_is_not_the_next_destination(irx):
    m, a, b = shared_tail(irx, tokens=3)
    c = m.open()
    m.extend(c, 3)
    d = m.fork(c)
    m.table
    pairs = [m.extend(a)]
    src = pairs[0][0]
    m.close(b)                                            # nobody holds the copied page any more
    pairs.append(m.extend(d))
    assert independent(pairs), pairs
    assert src not in m.table[d]
    free = m.free                                         # the table was read: the page is back
    m.close(c)
    assert m.free == free + 1


def test_extend_then_compact(irx):
    """The copy's source moves, its destination too."""
    m = irx.Pages(8, 4, 4, 4)
    filler = m.open()
    m.extend(filler, 12)                                  # pages 0 to 2
    a = m.open()
    m.extend(a, 3)                                        # page 3
    b = m.fork(a)
    m.table
    pair = m.extend(a)                                    # page 3 to page 4
    m.close(filler)
    moves = m.compact()
    assert len(moves) == 2 and independent([pair] + moves), (pair, moves)
    assert {int(p) for p in m.table.reshape(-1) if p >= 0} == {0, 1}
    assert {(pair[0], int(m.table[s, 0])) for s in (a, b)} == set(moves)


def test_a_copy_of_a_copy_reads_the_first_source(irx):
    """A move of a page whose own copy has not run yet takes its contents from where they are."""
    m, a, b = shared_tail(irx, pages=8, size=4, tokens=3)
    filler = m.open()
    m.extend(filler, 12)                                  # pages 1 to 3
    m.table
    pair = m.extend(a)                                    # page 0 to page 4
    m.close(filler)
    moves = m.compact()
    assert independent([pair] + moves), (pair, moves)
    now = int(m.table[a, 0])
    assert now == 1 and (0, 1) in moves


def test_when_only_pages_in_copies_are_left(irx):
    m, a, b = shared_tail(irx, pages=2, size=4, tokens=3)
    pair = m.extend(a)
    m.close(b)                                            # page 0 is free, but its copy may not have run
    c = m.open()
    with pytest.raises(irx.IrxError) as e:
        m.extend(c)
    assert e.value.code == 94 and m.length(c) == 0
    m.table                                               # the copy is queued by the time the table is used
    assert m.free == 1 and m.extend(c) is None and int(m.table[c, 0]) == pair[0]


def test_compaction_leaves_what_is_in_copies_and_a_later_one_finishes(irx):
    m, a, b = shared_tail(irx, pages=8, size=4, tokens=3)
    pair = m.extend(a)                                    # 0 to 1
    m.close(b)
    moves = m.compact()                                   # page 0 may not be written to yet
    assert independent([pair] + moves), (pair, moves)
    m.table
    moves = m.compact()
    assert moves == [(1, 0)] and int(m.table[a, 0]) == 0 and m.free == 7


@pytest.mark.parametrize("seed", range(24))
def test_gathered_copies_in_any_order(irx, seed):
    """Against a model that keeps each sequence's tokens. New tokens are written once the step's copies have
    run, in a random order or all at once from the pool as it was."""
    rng = random.Random(seed)
    pages, size, seqs, cols = rng.choice([7, 11, 24, 60]), rng.choice([1, 3, 4, 16]), 6, 9
    m = irx.Pages(pages, size, seqs, cols)
    pool, model, fresh, gathered = {}, {}, 0, 0
    for _ in range(150):
        pairs, pending = [], {}
        for _ in range(rng.randrange(1, 9)):
            op = rng.choice(["open", "extend", "extend", "extend", "fork", "close", "compact"])
            seq = rng.choice(list(model)) if model else None
            try:
                if op == "open":
                    model[m.open()] = []
                elif op == "compact":
                    pairs += m.compact()
                elif seq is None:
                    continue
                elif op == "extend":
                    n = rng.randrange(0, 2 * size + 1)
                    pair = m.extend(seq, n)
                    pairs += [pair] if pair else []
                    new = list(range(fresh, fresh + n))
                    fresh += n
                    pending.setdefault(seq, []).extend(zip(range(len(model[seq]), len(model[seq]) + n), new))
                    model[seq] = model[seq] + new
                elif op == "fork":
                    if seq not in pending:                # its tokens have been written
                        model[m.fork(seq)] = list(model[seq])
                else:
                    m.close(seq)
                    del model[seq]
                    pending.pop(seq, None)
            except irx.IrxError as e:
                assert e.code in (81, 94)
        assert independent(pairs), pairs
        gathered += len(pairs) > 1
        t = m.table
        was = dict(pool)
        for s, d in rng.sample(pairs, len(pairs)):
            for i in range(size):
                assert pool.get((s, i)) == was.get((s, i))
                pool[d, i] = pool.get((s, i))
        for seq, new in pending.items():
            for pos, tok in new:
                pool[int(t[seq, pos // size]), pos % size] = tok
        held = {int(p) for p in t.reshape(-1) if p >= 0}
        assert m.free == pages - len(held)
        for s, toks in model.items():
            assert m.length(s) == len(toks)
            assert [pool[int(t[s, j // size]), j % size] for j in range(len(toks))] == toks
    if pages > 11:
        assert gathered > 3
