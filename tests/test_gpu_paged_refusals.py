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
