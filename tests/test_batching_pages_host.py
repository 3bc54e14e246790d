"""The scheduler's count of pages against an engine that refuses what it has no pages for."""
import pytest

import batching
import eahmmf_b200 as eb
from test_paged_host import PagedEngine


class Strict(PagedEngine):
    """Returns EAHMMF_ST_CAPACITY, as the engine does."""

    def prefill_slot(self, slot, prompt, n_batch):
        self.len[slot] = len(prompt)
        if self.used() > self.n_pages:
            del self.len[slot]
            return eb.ST_CAPACITY, 0
        return 0, 1


@pytest.mark.parametrize("n_gen", [0, 1, 2])
@pytest.mark.parametrize("page", [16, 48])
def test_the_whole_prompt_is_counted(page, n_gen):
    b = batching.ContinuousBatcher(Strict(), n_slots=2, pages=2, page=page)
    with pytest.raises(ValueError):
        b.submit([1] * (2 * page + 1), n_gen)  # three pages
    first = b.submit([1] * page, 2)            # two pages while it runs
    later = b.submit([1] * (page + 1), n_gen)  # two: not beside it
    b.run()
    assert first.tokens == [1, 1] and len(later.tokens) == max(n_gen, 1) and not b.queue


@pytest.mark.parametrize("pages", [0, 4])
def test_a_refused_prefill_leaves_the_request_in_the_queue(pages):
    class Refusing(Strict):
        refuse = True

        def set_slots(self, n):
            return self.set_paged(n, 1 << 20, 16, "f16")

        def prefill_slot(self, slot, prompt, n_batch):
            return (eb.ST_CAPACITY, 0) if self.refuse else super().prefill_slot(slot, prompt, n_batch)

    e = Refusing()
    b = batching.ContinuousBatcher(e, n_slots=2, pages=pages, page=16)
    rs = [b.submit([1] * n, 3) for n in (5, 9)]
    for _ in range(2):
        with pytest.raises(RuntimeError):
            b.step()
        assert list(b.queue) == rs and not b.active and all(not r.tokens for r in rs)
    e.refuse = False
    b.run()
    assert [len(r.tokens) for r in rs] == [3, 3]
