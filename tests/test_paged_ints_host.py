"""Numbers that do not fit the C calls of the paged cache are refused, not taken modulo 2^32."""
import pytest

import eahmmf_b200 as eb

FAR = 1 << 32


@pytest.mark.parametrize("x", [FAR, FAR + 5, 1 << 31, -1, -FAR])
def test_pages_refuse_numbers_out_of_range(x):
    for a in range(4):
        args = [8, 16, 2, 4]
        args[a] = x
        with pytest.raises((ValueError, RuntimeError)):
            eb.Pages(*args)
    p = eb.Pages(8, 16, 2, 4)
    p.extend(0, 5)
    before = [t.tolist() for t in p.table()]
    for call in (lambda: p.extend(0, x + 5), lambda: p.extend(x, 5), lambda: p.extend(0, x), lambda: p.fork(x, 1), lambda: p.fork(0, x + 1),
                 lambda: p.truncate(x, 0), lambda: p.truncate(0, x), lambda: p.slide(x, 0), lambda: p.slide(0, x), lambda: p.slide(0, 0, x)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    assert [t.tolist() for t in p.table()] == before and p.free == 7 and p.refs(x) == -1
