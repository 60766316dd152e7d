"""GPU: calls of the paged operators that are refused, or that end early, without harm."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_list_that_shrinks_while_it_is_read():
    """An item's __index__ empties its list: the call sees what is left and is refused for unequal lengths."""
    from r4q import ops

    class Clears:
        def __init__(self, items):
            self.items = items

        def __index__(self):
            self.items.clear()
            return 0
    table = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    rows = []
    rows += [Clears(rows)] + [1] * 50
    with pytest.raises(ValueError, match="one length"):
        ops.kv_table_set(table, rows, list(range(51)), list(range(51)))
    assert rows == [] and not table.any()


def test_status_is_kept_or_taken():
    """clear=False leaves what was met, clear=True takes it; write and attention are both named."""
    from r4q import lib as L, ops
    k = torch.ones(1, 2, 128, dtype=torch.float16, device="cuda")
    pg = torch.zeros(2, 2, 16, 128, dtype=torch.uint8, device="cuda")
    bad = torch.tensor([[9]], dtype=torch.int32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.check_status()
    ops.paged_kv_write(k, k, pg, pg, bad, pos)
    ops.paged_flash_decode(k, pg, pg, bad, pos + 1)
    for clear in (False, False, True):
        with pytest.raises(L.R4QError, match="paged write and a paged attention") as e:
            ops.check_status(clear=clear)
        assert e.value.code == -6
    ops.check_status()


def test_status_of_calls_beside_a_thread_that_checks():
    """Of 200 bad calls each one is in a report: after a call has run, a check that begins later, or one that was under
    way, has named it."""
    import threading
    from r4q import lib as L, ops
    k = torch.ones(1, 1, 128, dtype=torch.float16, device="cuda")
    pg = torch.zeros(2, 1, 16, 128, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[9]], dtype=torch.int32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.check_status()
    stop, reports, checks, other = threading.Event(), [0], [0], []

    def check():
        while not stop.is_set():
            try:
                ops.check_status()
            except L.R4QError as e:
                if e.code == -6:
                    reports[0] += 1
                else:
                    other.append(e)
            checks[0] += 1
    t = threading.Thread(target=check)
    t.start()
    try:
        st = torch.cuda.Stream()
        for _ in range(200):
            before = reports[0]
            with torch.cuda.stream(st):
                ops.paged_kv_write(k, k, pg, pg, table, pos)
            st.synchronize()
            seen = checks[0]
            while checks[0] < seen + 2 and t.is_alive():
                pass
            assert reports[0] > before
    finally:
        stop.set()
        t.join()
    assert not other
    ops.check_status()
