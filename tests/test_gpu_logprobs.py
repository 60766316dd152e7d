"""GPU: log probabilities of given tokens with rank, entropy and top
alternatives (ops.token_logprobs) against 64-bit formulas.

Tolerances (u = 2^-24): the exponent (x - m) log2(e) of a term is rounded at
a magnitude of 64 at most where the term still counts, so a term is off by
2^-18 relative at most and so is their sum S; x_t - m and log S are rounded at
their own magnitudes and so is their difference: 2^-18 + 2 u (|x_t - m| + |log S|).
The entropy is log S - sum p (x - m): 2^-18 (1 + 2 sum p |x - m|) + 4 u of it.
Ids and ranks are whole numbers and equal (ties go to the lowest id)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def order(x):
    """Ids by (value, lowest id first), NaN last."""
    v = x.double().cpu().numpy()
    v = np.where(np.isnan(v), -np.inf, v) + 0.0
    last = np.isnan(x.double().cpu().numpy())
    return np.lexsort((np.arange(v.size), -v, last))


def check(x, tokens, k):
    from r4q import ops
    r = ops.token_logprobs(x, tokens, k)
    m = x.double().max(-1).values
    xd = x.double() - m[:, None]      # log softmax is the same from the maximum on; at 1e38 lse itself has no digit left for log S
    lse = torch.logsumexp(xd, -1)
    p = torch.softmax(xd, -1)
    t = torch.where(p > 0, xd, torch.zeros_like(xd))
    ent = lse - (p * t).sum(-1)
    spread = (p * t.abs()).sum(-1)
    assert (r.entropy.double() - ent).abs().le(2.0 ** -18 * (1 + 2 * spread) + 4 * U * ent.abs()).all()
    ids = np.stack([order(row) for row in x])
    assert np.array_equal(r.top_ids.cpu().numpy(), ids[:, :k])
    top = xd.gather(1, r.top_ids)
    fin = torch.isfinite(top)
    tol = 2.0 ** -18 + 2 * U * (top.abs() + lse.abs()[:, None])
    assert ((r.top_logprobs.double() - (top - lse[:, None])).abs() <= tol)[fin].all()
    assert (r.top_logprobs[~fin] == float("-inf")).all()
    if tokens is None:
        assert r.logprob is None and r.rank is None
        return r
    place = np.empty_like(ids)
    for row, i in zip(place, ids):
        row[i] = np.arange(i.size)
    assert np.array_equal(r.rank.cpu().numpy(), place[np.arange(len(place)), tokens.cpu().numpy()] + 1)
    xt = xd.gather(1, tokens[:, None])[:, 0]
    fin = torch.isfinite(xt)
    assert ((r.logprob.double() - (xt - lse)).abs() <= 2.0 ** -18 + 2 * U * (xt.abs() + lse.abs()))[fin].all()
    assert (r.logprob[~fin] == float("-inf")).all()
    return r


def logits(M, V, dtype, seed, std=2.5):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(M, V, generator=g, device="cuda") * std).to(dtype)
    return x, torch.randint(0, V, (M,), generator=g, device="cuda")


@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (1, 1, 0), (3, 7, 7), (2, 33, 32), (5, 1000, 20), (1, 151936, 20),
                                   (4, 32003, 5), (17, 50257, 32), (200, 4099, 1), (700, 513, 3), (2, 262145, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_vs_64_bits(M, V, k, dtype):
    x, t = logits(M, V, dtype, M + V)
    check(x, t, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties_take_the_lowest_id(dtype):
    for V in (40, 20000, 151936):
        x = torch.zeros(3, V, device="cuda", dtype=dtype)
        x[1] = (torch.arange(V, device="cuda") % 5).to(dtype)
        x[2, V // 2:] = -0.0                              # minus zero equals zero
        check(x, torch.tensor([V - 1, V // 3, V - 2], device="cuda"), 32)


@pytest.mark.parametrize("V", [5000, 151936])
@pytest.mark.parametrize("step", [1, 2, 8, 512, 1024, 2048, 4096])
def test_largest_values_in_one_place(V, step):
    """The 40 largest values next to one another, or apart by powers of two, rising and falling."""
    x, _ = logits(4, V, torch.float16, step, std=1.0)
    at = (torch.arange(40, device="cuda") * step + 3) % V
    n = torch.arange(40, device="cuda").half()
    x[0, at] = 20 + n
    x[1, at] = 70 - n
    x[2, at] = 30
    x[3, at] = float("-inf")
    check(x, at[torch.tensor([0, 39, 20, 7], device="cuda")], 32)


def test_sorted_rows():
    for V in (3000, 70000):
        x = torch.linspace(-30, 30, V, device="cuda").repeat(2, 1)
        x[1] = x[1].flip(0)
        check(x, torch.tensor([V - 1, V // 2], device="cuda"), 20)


def test_masked_rows_and_extremes():
    """-inf masks that leave 1 or 3 ids, the type's lowest value as a mask, huge and tiny spreads."""
    x, t = logits(6, 9000, torch.float32, 5)
    x[0] = float("-inf")
    x[0, 77] = 3.0
    x[1, 3:] = float("-inf")
    x[2] = torch.finfo(torch.float32).min
    x[2, 5000] = 1.0
    x[3] *= 1e30
    x[4] = 1e-30
    x[5] = torch.finfo(torch.float32).min
    t[0], t[1] = 77, 1
    r = check(x, t, 8)
    assert r.logprob[0] == 0 and r.entropy[0] == 0
    h, th = logits(3, 9000, torch.float16, 6)
    h[0] = torch.finfo(torch.float16).min
    h[1] = torch.finfo(torch.float16).max
    h[2, 1:] = float("-inf")
    check(h, th, 32)


def test_rows_that_are_no_distribution():
    from r4q import ops
    V = 5001
    x, t = logits(5, V, torch.float16, 9)
    x[0] = float("-inf")
    x[1, 4000] = float("nan")
    x[2, 10] = float("inf")
    x[3] = float("nan")
    t[1] = 5
    r = ops.token_logprobs(x, t, 4)
    for out in (r.logprob, r.entropy, r.top_logprobs[:, 0], r.top_logprobs[:, 3]):
        assert torch.isnan(out[:4]).all() and torch.isfinite(out[4])
    want = [order(row)[:4].tolist() for row in x]
    assert r.top_ids.tolist() == want and want[0] == want[3] == [0, 1, 2, 3] and want[2][0] == 10
    assert r.rank[1] == 1 + int((x[1] > x[1, 5]).sum() + (x[1, :5] == x[1, 5]).sum())


def test_tokens_outside_and_none():
    from r4q import ops
    x, t = logits(4, 800, torch.float16, 2)
    t[0], t[1] = -1, 800
    r = ops.token_logprobs(x, t, 2)
    assert torch.isnan(r.logprob[:2]).all() and (r.rank[:2] == 0).all() and torch.isfinite(r.entropy).all()
    assert torch.isfinite(r.logprob[2:]).all()
    check(x, None, 5)
    empty = ops.token_logprobs(x[:0], t[:0], 3)
    assert empty.top_ids.shape == (0, 3) and empty.logprob.shape == (0,)


def test_strides_and_alignment():
    """Rows of any stride from any element on, and columns apart (copied by the wrapper)."""
    for dtype in (torch.float16, torch.float32):
        big, t = logits(6, 10007, dtype, 3)
        for off in range(1, 9):
            check(big[:, off:off + 9990], t % 9990, 6)
        check(big[::2], t[::2], 6)
        check(big.t()[:3000].t(), t % 3000, 6)


def test_rows_beyond_32_bit_offsets_and_grids():
    """Rows whose first element lies beyond 2^31, and more rows than a grid dimension takes."""
    from r4q import ops
    V = 1 << 20
    x = torch.zeros(2100, V, dtype=torch.float16, device="cuda")
    big, t = logits(3, V, torch.float16, 7)
    x[-3:] = big
    t = torch.cat([torch.zeros(2097, dtype=torch.int64, device="cuda"), t])
    r = ops.token_logprobs(x, t, 3)
    few = check(big, t[-3:], 3)
    # the sums run in an order that goes by the number of rows, so both lie within the bound of the exact value
    # (here |x_t - m| and log S below 32): twice that of each other; ids and ranks are equal
    assert torch.equal(r.rank[-3:], few.rank) and torch.equal(r.top_ids[-3:], few.top_ids)
    for a, b, tol in ((r.logprob, few.logprob, 1), (r.top_logprobs, few.top_logprobs, 1), (r.entropy, few.entropy, 64)):
        assert ((a[-3:] - b).abs() <= 2 * tol * (2.0 ** -18 + 2 * U * 64)).all()
    assert (r.rank[:2097] == 1).all() and torch.equal(r.top_ids[:2097], torch.arange(3, device="cuda").expand(2097, 3))
    del x, r
    many, t = logits(70000, 40, torch.float32, 8)
    check(many, t, 2)


def test_repeatable_streams_and_graphs():
    from r4q import ops
    sets = [logits(5, 151936, torch.float16, 31), logits(300, 32003, torch.bfloat16, 32)]
    first = [ops.token_logprobs(*s, 20) for s in sets]
    torch.cuda.synchronize()
    graphs, outs, cap = [], [], torch.cuda.Stream()
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            outs.append(ops.token_logprobs(*s, 20))
        graphs.append(g)
    streams, eager = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
                eager[1 - i].append(ops.token_logprobs(*sets[1 - i], 20))
    torch.cuda.synchronize()
    for i in (0, 1):
        for other in (outs[i], *eager[i]):
            assert all(torch.equal(a, b) for a, b in zip(first[i], other))


def test_wrapper_refusals_on_device_tensors():
    from r4q import ops
    x, t = logits(2, 50, torch.float16, 1)
    for call in (lambda: ops.token_logprobs(x.double(), t), lambda: ops.token_logprobs(x[0], t),
                 lambda: ops.token_logprobs(x, t.int()), lambda: ops.token_logprobs(x, t[:1]),
                 lambda: ops.token_logprobs(x, t, 51), lambda: ops.token_logprobs(x, t, 33),
                 lambda: ops.token_logprobs(x, t, -1)):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_served_requests_carry_likelihoods():
    """BatchedEngine over the decode context: each generated token's likelihood, rank, entropy and alternatives equal
    those of the logits it was sampled from; requests that ask for none get none, and the tokens do not change."""
    from r4q import decode, ops, serve
    from test_gpu_serve import CFG, RecordingBackend, _model
    m = _model(3)

    class Rec(RecordingBackend):
        def logprobs(self, lg, toks, k):
            return self.be.logprobs(lg, toks, k)

    def run(lp):
        rec = Rec(serve.SlotBackend(m, CFG, batch=3))
        eng = serve.BatchedEngine(rec)
        rec.eng = eng
        reqs = [eng.submit([3, 5, 7], max_new_tokens=4, logprobs=lp[0]),
                eng.submit([9], max_new_tokens=5, temperature=0.8, top_p=0.9, seed=4, logprobs=lp[1]),
                eng.submit([1, 2], max_new_tokens=3)]
        eng.run()
        return reqs, rec
    plain, _ = run((None, None))
    reqs, rec = run((5, 0))
    assert [r.tokens for r in reqs] == [r.tokens for r in plain]
    assert reqs[2].token_logprobs == [] and plain[0].token_logprobs == []
    for r, k in zip(reqs[:2], (5, 0)):
        assert [x.token for x in r.token_logprobs] == r.tokens
        for x, lg in zip(r.token_logprobs, rec.seen[r.id]):
            ref = torch.log_softmax(lg.double(), -1)
            ids = order(lg)
            assert abs(x.logprob - ref[x.token].item()) < 1e-5 and len(x.top) == k
            assert ids[x.rank - 1] == x.token and [i for i, _ in x.top] == ids[:k].tolist()
            assert abs(x.entropy + (ref.exp() * ref).sum().item()) < 1e-4
    ops.check_status()
    decode.clear_contexts()
