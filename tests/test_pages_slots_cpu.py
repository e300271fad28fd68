"""Steps of slots that nobody holds take no pages."""
import pytest

from test_pages_cpu import consistent, make


def test_a_slot_that_is_not_in_use_takes_no_pages():
    c = make(states=({}, {}))
    a, b = c.acquire(), c.acquire()
    c.extend(a, 0, 9)
    c.release(b)
    free = c.free_pages()
    for slot in (b, -1, c.slots, 5):
        with pytest.raises(ValueError):
            c.extend(slot, 0, 9)
        with pytest.raises(ValueError):
            c.extend_all([a, slot], 0, 9)
        with pytest.raises(ValueError):
            c.truncate(slot, 0)
        consistent(c)
        assert c.free_pages() == free and c.lengths[a] == 9
    # and the next one to take the slot starts with none
    again = c.acquire()
    assert c.held[again] == [] and c.lengths[again] == 0
    c.extend_all([again], 0, 17)
    assert len(c.held[again]) == 3
    consistent(c)
