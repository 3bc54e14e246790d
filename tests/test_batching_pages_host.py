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
