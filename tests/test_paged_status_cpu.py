"""What the status words of the paged and likelihood kernels are reported as (host code alone)."""
import itertools

from r4q import lib as L

TIMEOUT, PAGE = 1, 2


def test_every_condition_is_named_and_a_timeout_gives_the_code():
    for w, a, k in itertools.product((0, PAGE), (0, TIMEOUT, PAGE, TIMEOUT | PAGE), (0, TIMEOUT)):
        st, text = L.LIB.r4q_debug_status_of(w, a, k), L.last_error()
        late, bad = (a | k) & TIMEOUT, (w | a) & PAGE
        assert st == (-5 if late else -6 if bad else 0), (w, a, k)
        if not st:
            continue
        assert ("gave up" in text) == bool(late) and ("outside the cache" in text) == bool(bad), text
        waits, _, pages = text.partition("; ") if late else ("", "", text)
        assert ("paged attention" in waits) == bool(a & TIMEOUT) and ("likelihood" in waits) == bool(k & TIMEOUT), text
        assert ("paged write" in pages) == bool(w & PAGE) and ("paged attention" in pages) == bool(a & PAGE), text
