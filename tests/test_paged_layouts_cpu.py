"""Page tensors whose pages do not lie one behind the other are refused before
anything is launched (CPU: the layout is looked at before the device)."""
import pytest
import torch

from r4q import ops

K = torch.zeros(2, 2, 128, dtype=torch.float16)
TABLE, POS = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
PAGES = torch.zeros(4, 2, 16, 128, dtype=torch.uint8)


@pytest.mark.parametrize("bad", [
    torch.zeros(1, 2, 16, 128, dtype=torch.uint8).expand(4, 2, 16, 128),                 # one page, four times
    torch.zeros(3 * 2048 + 4096, dtype=torch.uint8).as_strided((4, 2, 16, 128), (2048, 2048, 128, 1)),   # overlapping
])
def test_pages_on_top_of_one_another_are_refused(bad):
    for kp, vp in ((bad, PAGES), (PAGES, bad), (bad, bad)):
        with pytest.raises(ValueError, match="behind"):
            ops.paged_flash_decode(K, kp, vp, TABLE, POS)
        with pytest.raises(ValueError, match="behind"):
            ops.paged_kv_write(K, K, kp, vp, TABLE, POS)


def test_layouts_that_are_pages_pass_on_to_the_device_check():
    both = torch.zeros(4, 2, 2, 16, 128, dtype=torch.uint8)
    one = torch.zeros(1, 2, 16, 128, dtype=torch.uint8)
    for kp, vp in ((PAGES, PAGES), (both[:, 0], both[:, 1]), (PAGES[::2], PAGES[1::2]), (one, one)):
        with pytest.raises(ValueError, match="CUDA"):
            ops.paged_flash_decode(K, kp, vp, TABLE, POS)
        with pytest.raises(ValueError, match="CUDA"):
            ops.paged_kv_write(K, K, kp, vp, TABLE, POS)


def test_a_table_cell_twice_is_refused():
    """The kernel writes the cells in any order."""
    import ctypes as C
    import random
    from r4q import lib as L

    def put(cells):
        r, c = ((C.c_int * len(cells))(*x) for x in zip(*cells))
        return L.LIB.r4q_kv_table_set(C.c_void_p(256), 50, 60, 50, r, c, r, len(cells), None)   # refused before any launch
    many = [(i, j) for i in range(60) for j in range(50)]
    random.Random(1).shuffle(many)
    for cells in ([(0, 0), (0, 0)], [(1, 2), (2, 1), (1, 2)], many + [many[7]]):
        assert put(cells) == -1 and "twice" in L.last_error()


@pytest.mark.parametrize("kw", ["k_caches", "v_caches", "k_scales", "v_scales"])
def test_prefill_into_pages_refuses_what_it_would_ignore(kw):
    from r4q import paged, prefill
    pages = paged.PagedKVCache(1, 4, 2, 16, 1, 4, "cpu")
    with pytest.raises(ValueError, match=kw):
        prefill.prefill_logits(*[None] * 25, pages=pages, **{kw: [torch.ones(2)]})
