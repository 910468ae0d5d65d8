"""GPU checks of paged attention where queries are not finite beside sinks."""

import numpy as np
import pytest

from tests._packed import Dev
from tests._paged import attend
from tests.test_gpu_paged import Attend, done, say

pytestmark = pytest.mark.gpu

# of several workgroups' shapes, cut into spans and not
CALLS = [
    (64, 8, 64, [1], [5000]), (32, 4, 128, [1, 1, 7], [900, 2000, 40]), (64, 8, 64, [100], [8000]), (32, 4, 128, [250], [3000]),
    (64, 1, 128, [500], [11]), (64, 8, 64, [500, 1, 3, 20], [2500, 60, 700, 300]), (32, 4, 128, [300, 20, 1], [1500, 900, 2000])]


def some_rows(a, rows):
    return {int(r): range(a.nh) for r in rows}


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", CALLS)
def test_queries_not_finite_beside_sinks(tg, nh, nkv, hd, lens, past, bad):
    """All rows of the first sequence, or four that fill a wave's places: NaN in every head, whatever the sinks add, also where
    their own positions' blocks are NaN; the other rows are what they are without them."""
    for rows in (range(lens[0]), range(4, 8)):
        if rows[-1] >= lens[0]:
            continue
        rows = list(rows)
        for blocks in (False, True):
            say(f"attention {nh, nkv, hd, lens, past} rows {rows[:1]}.. q={bad} blocks={blocks}")
            a = Attend(41, nh, nkv, hd, lens, past, 32, sinks=True)
            a.q[rows, 5::hd] = bad
            if blocks:   # as the append of such rows leaves them: later rows of the sequence are NaN, too
                for j in range((past[0] + rows[0]) // 16, (past[0] + rows[-1]) // 16 + 1):
                    a.pages.ek[a.pages.table[0, 16 * j // 32], :, 16 * j % 32 // 16] = 255
            dev = Dev(tg)
            a.call(dev)
            done(tg)
            got = dev.read(a.out, a.q)
            assert np.isnan(got[rows]).all(), int((~np.isnan(got[rows])).sum())
            gone = lens[0] if blocks else len(rows)
            rest = [r for r in range(a.rows) if r not in rows and (not blocks or r >= gone)]
            rest = sorted({*rest[:2], *rest[len(rest) // 2:len(rest) // 2 + 1], *rest[-2:]})
            if rest:
                want, tol = attend(a.q, a.pages, a.cu, lens, past, nh, sinks=a.sinks, only=some_rows(a, rest))
                assert np.all(np.abs(got[rest] - want[rest]) <= tol[rest])
            dev.free()
