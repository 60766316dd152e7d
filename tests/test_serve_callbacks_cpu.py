"""A callback or a backend that raises in the middle of a step (CPU, stand-in
backend): the rows that were not served yet are decoded again, with the draws
they would have had, and every token has one likelihood beside it."""
import pytest
import torch

from r4q import serve

V = 11


class Backend:
    """Logits are a function of (token, position): a repeated step repeats them."""
    batch, max_seq = 2, 32

    def __init__(self):
        self.fail = 0

    def _row(self, tok, pos):
        return 2 * torch.randn(V, generator=torch.Generator().manual_seed(100 * tok + pos))

    def prefill(self, slot, prompt):
        return self._row(prompt[-1], len(prompt) - 1)

    def step(self, tokens, positions):
        return torch.stack([self._row(t, p) for t, p in zip(tokens, positions)])

    def logprobs(self, logits, tokens, k):
        if self.fail:
            self.fail -= 1
            raise RuntimeError("no likelihoods")
        lp = torch.log_softmax(logits, -1)
        return [serve.TokenLogprob(t, float(r[t]), 1, 0.0, tuple((i, float(r[i])) for i in r.topk(k).indices.tolist()))
                for t, r in zip(tokens, lp)]


A = dict(prompt=[1], max_new_tokens=4)
B = dict(prompt=[2], max_new_tokens=6, temperature=1.5, seed=3)


def alone(kw):
    r, = serve.BatchedEngine(Backend()).generate([kw["prompt"]], **{k: v for k, v in kw.items() if k != "prompt"})
    return r


def run(a, b, raise_at=None, fail_at=None):
    """Both requests; a's callback raises at its token number `raise_at`, or the backend's `fail_at`-th step has no likelihoods."""
    be, raised = Backend(), []

    def on_token(r, tok):
        if len(r.tokens) == raise_at:
            raised.append(tok)
            raise RuntimeError("callback")
    eng = serve.BatchedEngine(be)
    ra, rb = eng.submit(**a, on_token=on_token), eng.submit(**b)
    n = 0
    while eng.queue or eng.active:
        n += 1
        be.fail = n == fail_at
        try:
            eng.step()
        except RuntimeError as e:
            raised.append(e)
    assert raised
    return ra, rb


@pytest.mark.parametrize("a_lp", [None, 1])
@pytest.mark.parametrize("b", [B, dict(B, logprobs=0), dict(B, logprobs=2, temperature=0.0)])
def test_a_raising_callback_leaves_the_other_rows_as_they_were(a_lp, b):
    ra, rb = run(dict(A, logprobs=a_lp), b, raise_at=2)
    want = alone(b)
    assert rb.tokens == want.tokens and rb.token_logprobs == want.token_logprobs
    assert [x.token for x in ra.token_logprobs] == (ra.tokens if a_lp else [])


@pytest.mark.parametrize("lp", [None, 1])
def test_a_callback_of_a_sampled_row_that_asks_for_likelihoods(lp):
    """The row whose own callback raises keeps its draw, the one behind it does not."""
    a = dict(A, temperature=1.2, seed=9, logprobs=1)
    ra, rb = run(a, dict(B, logprobs=lp), raise_at=2)
    assert rb.tokens == alone(B).tokens
    assert ra.tokens[:2] == alone(a).tokens[:2] and [x.token for x in ra.token_logprobs] == ra.tokens


@pytest.mark.parametrize("fail_at", [1, 3])
def test_a_step_without_likelihoods_is_repeated_as_it_was(fail_at):
    """Also an admission (step 1): the request waits again."""
    a, b = dict(A, temperature=1.2, seed=9, logprobs=1), dict(B, logprobs=2)
    ra, rb = run(a, b, fail_at=fail_at)
    for r, kw in ((ra, a), (rb, b)):
        want = alone(kw)
        assert r.tokens == want.tokens and r.token_logprobs == want.token_logprobs


def test_backend_with_more_rows_than_the_engine_has_slots():
    """Its logits carry rows of no request: they are not handed to the likelihoods."""
    class Wide(Backend):
        def step(self, tokens, positions):
            return torch.cat([super().step(tokens, positions), torch.zeros(2, V)])

        def logprobs(self, logits, tokens, k):
            assert logits.shape[0] == len(tokens)
            return super().logprobs(logits, tokens, k)
    r, = serve.BatchedEngine(Wide(), batch=1).generate([[1]], max_new_tokens=4, logprobs=2)
    want = alone(dict(A, logprobs=2))
    assert r.tokens == want.tokens and r.token_logprobs == want.token_logprobs
