"""GPU: the bounded waits of the paged attention and the likelihood kernel.  A
poll limit of 0 makes every wait give up before it looks; the kernels then wait
for their copies, return, and report it, and the next call is right."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_polls():
    from r4q import lib as L, ops
    ops.check_status()

    class Limit:
        def __enter__(self):
            self.old = L.LIB.r4q_debug_wait_limit(0)

        def __exit__(self, *a):
            torch.cuda.synchronize()
            assert L.LIB.r4q_debug_wait_limit(-1) == 0 and self.old == 1 << 22
    yield Limit()
    assert L.LIB.r4q_debug_wait_limit(-1) == 1 << 22


@pytest.mark.parametrize("lens,blocks", [([300, 1], 20), ([3000, 17, 0], 200), ([40000] * 20, 2500)])
def test_attention_gives_up_and_recovers(no_polls, lens, blocks):
    """A table that one kernel serves, and tables of two kernels, the last with tiles in every warp."""
    from r4q import lib as L, ops
    g = torch.Generator("cuda").manual_seed(1)
    pg = torch.randint(0x20, 0x48, (2, 64, 2, 16, 128), generator=g, device="cuda", dtype=torch.uint8)
    q = torch.randn(len(lens), 16, 128, generator=g, device="cuda").half()
    table = torch.randint(0, 64, (len(lens), blocks), generator=g, device="cuda", dtype=torch.int32)
    seq = torch.tensor(lens, device="cuda")
    want = ops.paged_flash_decode(q, pg[0], pg[1], table, seq)
    ops.check_status()
    with no_polls:
        ops.paged_flash_decode(q, pg[0], pg[1], table, seq)
    with pytest.raises(L.R4QError, match="paged attention") as e:
        ops.check_status()
    assert e.value.code == -5
    assert torch.equal(ops.paged_flash_decode(q, pg[0], pg[1], table, seq), want)
    ops.check_status()


@pytest.mark.parametrize("M,V,k,dtype", [(1, 151936, 20, torch.float16), (3, 5000, 0, torch.bfloat16),
                                         (700, 40000, 5, torch.float32)])
def test_likelihoods_give_up_and_recover(no_polls, M, V, k, dtype):
    """A cluster for a row, and a CTA for a row; the rows of a call that gave up are NaN."""
    from r4q import lib as L, ops
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn(M, V, generator=g, device="cuda").to(dtype)
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    want = ops.token_logprobs(x, t, k)
    ops.check_status()
    with no_polls:
        r = ops.token_logprobs(x, t, k)
    assert torch.isnan(r.logprob).all() and torch.isnan(r.entropy).all() and torch.isnan(r.top_logprobs).all()
    with pytest.raises(L.R4QError, match="likelihood") as e:
        ops.check_status()
    assert e.value.code == -5
    assert all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(x, t, k), want))
    ops.check_status()


def test_a_bad_page_beside_a_wait_that_gave_up(no_polls):
    from r4q import lib as L, ops
    k = torch.ones(1, 2, 128, dtype=torch.float16, device="cuda")
    pg = torch.zeros(2, 2, 16, 128, dtype=torch.uint8, device="cuda")
    bad = torch.tensor([[9]], dtype=torch.int32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.paged_kv_write(k, k, pg, pg, bad, pos)
    with no_polls:
        ops.paged_flash_decode(k, pg, pg, bad.zero_(), pos + 1)
    with pytest.raises(L.R4QError, match="gave up.*paged write") as e:
        ops.check_status()
    assert e.value.code == -5
    ops.check_status()
