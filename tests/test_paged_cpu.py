"""Paged cache on the CPU: the page bookkeeping (r4q.paged.PageAllocator)
against a model of the cache as plain lists of values, and the refusals of
the C entry points and of the tensor wrappers, none of which reaches a GPU."""
import ctypes as C
import random
import struct

import pytest
import torch

from r4q import lib as L
from r4q import ops, paged, serve


class Mirror:
    """The pool as a list of pages of values, written through the table that
    the plans leave; checks each plan as it carries it out."""

    def __init__(self, a):
        self.a = a
        self.pool = [[None] * a.page for _ in range(a.n_pages)]
        self.table = [[0] * a.max_blocks for _ in range(a.seqs)]

    def run(self, plan):
        assert len(set(plan.dst)) == len(plan.dst) and not set(plan.src) & set(plan.dst)
        for s, d in zip(plan.src, plan.dst):
            self.pool[d] = list(self.pool[s])
        cells = list(zip(plan.rows, plan.cols))
        assert len(set(cells)) == len(cells)
        for (r, c), v in zip(cells, plan.values):
            self.table[r][c] = v

    def write(self, seq, pos, value):
        page = self.table[seq][pos // self.a.page]
        assert self.a.refs[page] == 1, "a shared page was written"
        self.pool[page][pos % self.a.page] = value

    def read(self, seq, n):
        return [self.pool[self.table[seq][p // self.a.page]][p % self.a.page] for p in range(n)]


def invariants(a):
    held = [p for b in a.blocks for p in b]
    assert all(a.refs[p] == held.count(p) for p in range(a.n_pages))
    assert sorted(a.free_pages) == [p for p in range(a.n_pages) if a.refs[p] == 0]
    assert all(len(b) == -(-n // a.page) for b, n in zip(a.blocks, a.lengths))


@pytest.mark.parametrize("page,pages,seed", [(16, 12, 1), (16, 40, 2), (32, 9, 3), (48, 25, 4)])
def test_random_operations_keep_every_sequence_intact(page, pages, seed):
    rng = random.Random(seed)
    a = paged.PageAllocator(pages, page, 6, 8)
    mir, want, tick = Mirror(a), [[] for _ in range(6)], 0
    refused = 0
    for _ in range(400):
        op, s = rng.choice("eeeefFc"), rng.randrange(6)
        if op == "e":
            counts = {t: rng.randrange(0, 2 * page) for t in rng.sample(range(6), rng.randrange(1, 4))}
            before = ([list(b) for b in a.blocks], list(a.lengths), list(a.refs), list(a.free_pages))
            try:
                mir.run(a.extend(counts))
            except (paged.OutOfPages, ValueError):
                refused += 1
                assert before == (a.blocks, a.lengths, a.refs, a.free_pages)
                continue
            for t, n in counts.items():
                for _ in range(n):
                    tick += 1
                    mir.write(t, len(want[t]), tick)
                    want[t].append(tick)
        elif op == "f":
            mir.run(a.free(s))
            want[s] = []
        elif op == "F":
            t = rng.randrange(6)
            if want[t] or t == s:
                continue
            n = rng.randrange(len(want[s]) + 1)
            mir.run(a.fork(s, t, n))
            want[t] = want[s][:n]
        else:
            mir.run(a.compact())
            used = pages - a.free_count
            assert all(a.refs[p] for p in range(used)) and not any(a.refs[used:])
        invariants(a)
        for t in range(6):
            assert mir.read(t, len(want[t])) == want[t], (op, t)
    assert refused and tick > 100


def test_two_forks_writing_one_page_copy_it_once():
    a = paged.PageAllocator(4, 16, 2, 4)
    a.extend({0: 5})
    a.fork(0, 1)
    plan = a.extend({0: 1, 1: 1})                 # the first writer copies, the second keeps the page
    assert (plan.src, plan.dst, a.refs[:2]) == ([0], [1], [1, 1])


def test_check_writable():
    a = paged.PageAllocator(8, 16, 3, 4)
    a.extend({0: 40})
    a.check_writable(0, 40)
    a.fork(0, 1, 20)
    for seq, end in ((0, 41), (0, 1), (1, 20), (3, 1), (-1, 1)):
        with pytest.raises(ValueError):
            a.check_writable(seq, end)
    a.check_writable(2, 0)
    a.free(0)
    a.check_writable(1, 20)


def test_check_writable_from_a_position():
    a = paged.PageAllocator(8, 16, 2, 4)
    a.extend({0: 40})
    a.fork(0, 1, 20)                              # pages 0 and 1 are shared, 2 is not
    a.check_writable(0, 40, 39)
    a.check_writable(0, 33, 32)
    for end, start in ((32, 31), (33, 31), (1, 0), (41, 40)):
        with pytest.raises(ValueError):
            a.check_writable(0, end, start)
    a.extend({1: 1})
    a.check_writable(1, 21, 20)


def test_allocator_refusals():
    a = paged.PageAllocator(4, 16, 3, 2)
    a.extend({0: 20})
    with pytest.raises(ValueError):
        a.extend({0: 13})                         # beyond max_blocks
    with pytest.raises(paged.OutOfPages):
        a.extend({1: 32, 2: 16})
    with pytest.raises(ValueError):
        a.extend({3: 1})
    with pytest.raises(ValueError):
        a.extend({0: -1})
    with pytest.raises(ValueError):
        a.fork(0, 1, 21)
    a.extend({1: 1})
    with pytest.raises(ValueError):
        a.fork(0, 1)                              # not empty
    with pytest.raises(ValueError):
        a.free(-1)
    for bad in [(0, 16, 1, 1), (1, 8, 1, 1), (1, 24, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)]:
        with pytest.raises(ValueError):
            paged.PageAllocator(*bad)


# r4q_paged_cache in the platform's C layout
PAGED_CACHE = struct.Struct("@PPlliiiPliiPP")
P16 = C.c_void_p(256)                             # never dereferenced: validation fails first


def cache(**kw):
    d = dict(k_pages=256, v_pages=256, k_stride=0, v_stride=0, n_pages=4, page=16, Hk=2, table=256, ld_table=4, seqs=3,
             max_blocks=4, k_scale=0, v_scale=0)
    d.update({k: v or 0 for k, v in kw.items()})
    return PAGED_CACHE.pack(*d.values())


def attn(c=None, q=P16, ldq=512, seq=P16, o=P16, ldo=512, B=2, H=4, flags=0, ws=P16, ws_bytes=1 << 40):
    return L.LIB.r4q_paged_flash_decode(q, ldq, c or cache(), seq, o, ldo, B, H, flags, ws, ws_bytes, None)


def write(c=None, q=None, ldq=512, k=P16, ldk=256, v=P16, ldv=256, qw=None, kw=None, cos=None, sin=None, ts=64, tr=0,
          qo=None, ldqo=512, ko=None, ldko=256, rows=None, pos=P16, M=2, H=0, flags=0):
    return L.LIB.r4q_paged_kv_write(q, ldq, k, ldk, v, ldv, qw, kw, cos, sin, ts, tr, qo, ldqo, ko, ldko,
                                    c or cache(), rows, pos, M, H, 1e-6, flags, None)


BAD_CACHES = [(dict(page=8), -1), (dict(page=40), -1), (dict(page=0), -1), (dict(n_pages=0), -1), (dict(Hk=0), -1),
              (dict(seqs=0), -1), (dict(max_blocks=0), -1), (dict(ld_table=3), -1), (dict(k_pages=None), -1),
              (dict(v_pages=None), -1), (dict(table=None), -1), (dict(k_stride=4000), -1), (dict(k_stride=4104), -2),
              (dict(v_pages=264), -2), (dict(max_blocks=1 << 27, ld_table=1 << 27), -1)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches_refused(kw, code):
    assert attn(cache(**kw)) == code and "paged_flash_decode" in L.last_error()
    assert write(cache(**kw)) == code and "paged_kv_write" in L.last_error()


@pytest.mark.parametrize("kw,code", [(dict(q=None), -1), (dict(o=None), -1), (dict(seq=None), -1), (dict(B=-1), -1),
                                     (dict(B=4), -1), (dict(H=3), -1), (dict(H=1), -1), (dict(flags=2), -1),
                                     (dict(ldq=511), -1), (dict(ldo=504), -1), (dict(q=C.c_void_p(264)), -2),
                                     (dict(ldq=516), -2), (dict(o=C.c_void_p(2)), -2)])
def test_attention_refusals(kw, code):
    assert attn(**kw) == code and "paged_flash_decode" in L.last_error()


def test_empty_calls_are_no_calls():
    assert attn(B=0, q=None, o=None, seq=None) == 0
    assert write(M=0, k=None, v=None, pos=None) == 0
    assert L.LIB.r4q_kv_copy_pages(P16, 2, 64, 16, 16, 4, None, None, 0, None) == 0
    assert L.LIB.r4q_kv_table_set(P16, 4, 4, 4, None, None, None, 0, None) == 0
    assert L.LIB.r4q_token_logprobs(P16, 0, 8, None, 0, 8, 0, None, None, None, None, None, None) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(pos=None), -1), (dict(M=-1), -1), (dict(M=4), -1),
    (dict(q=P16, H=4), -1), (dict(flags=1), -1), (dict(flags=2), -1), (dict(flags=4), -1), (dict(flags=16), -1),
    (dict(flags=1, q=P16, H=4, qo=P16, kw=P16), -1), (dict(flags=2, cos=P16, sin=P16, tr=0), -1),
    (dict(flags=2, cos=P16, sin=P16, tr=9, ts=32), -1), (dict(ldk=248), -1), (dict(ko=P16, ldko=8), -1),
    (dict(ldk=260), -2), (dict(k=C.c_void_p(264)), -2), (dict(flags=2, cos=P16, sin=C.c_void_p(8), tr=9), -2),
    (dict(flags=1, kw=C.c_void_p(8)), -2)])
def test_write_refusals(kw, code):
    assert write(**kw) == code and "paged_kv_write" in L.last_error()


def ints(*v):
    return (C.c_int * len(v))(*v)


@pytest.mark.parametrize("src,dst,code", [((0,), (4,), -1), ((-1,), (1,), -1), ((0, 1), (2, 2), -1),
                                          ((0, 1), (1, 2), -1), ((3,), (3,), -1)])
def test_copy_refusals(src, dst, code):
    st = L.LIB.r4q_kv_copy_pages(P16, 2, 4096, 1024, 1024, 4, ints(*src), ints(*dst), len(src), None)
    assert st == code and "kv_copy_pages" in L.last_error()


def test_copy_and_table_layout_refusals():
    def one(pool=P16, outer=2, os=4096, ps=1024, pb=1024):
        return L.LIB.r4q_kv_copy_pages(pool, outer, os, ps, pb, 4, ints(0), ints(1), 1, None)
    assert one(pool=None) == -1 and one(ps=512) == -1 and one(outer=70000) == -1 and one(pb=0) == -1
    assert one(pool=C.c_void_p(264)) == -2 and one(os=4104) == -2 and one(ps=1032) == -2
    for r, c in ((4, 0), (-1, 0), (0, 3), (0, -1)):
        assert L.LIB.r4q_kv_table_set(P16, 4, 4, 3, ints(r), ints(c), ints(7), 1, None) == -1
    assert L.LIB.r4q_kv_table_set(P16, 2, 4, 3, ints(0), ints(0), ints(7), 1, None) == -1


@pytest.mark.parametrize("kw,code", [(dict(V=0), -1), (dict(k=33), -1), (dict(k=-1), -1), (dict(V=8, ld=8, k=9), -1),
                                     (dict(M=-1), -1), (dict(type=3), -1), (dict(x=None), -1), (dict(ld=99), -1),
                                     (dict(tokens=None), -1), (dict(x=C.c_void_p(257)), -2),
                                     (dict(x=C.c_void_p(258), type=2), -2)])
def test_logprob_refusals(kw, code):
    d = dict(x=P16, type=0, ld=100, tokens=P16, M=2, V=100, k=5)
    d.update(kw)
    st = L.LIB.r4q_token_logprobs(d['x'], d['type'], d['ld'], d['tokens'], d['M'], d['V'], d['k'], P16, P16, P16, P16,
                                  P16, None)
    assert st == code and "token_logprobs" in L.last_error()


def test_wrappers_take_cuda_tensors_only_and_host_lists():
    k = torch.zeros(2, 2, 128, dtype=torch.float16)
    pg = torch.zeros(4, 2, 16, 128, dtype=torch.uint8)
    t, pos = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.paged_kv_write(k, k, pg, pg, t, pos), lambda: ops.paged_flash_decode(k, pg, pg, t, pos),
                 lambda: ops.kv_copy_pages(pg, [0], [1]), lambda: ops.kv_table_set(t, [0], [0], [1]),
                 lambda: ops.token_logprobs(k[0], pos, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: ops.paged_flash_decode(None, pg, pg, t, pos), lambda: ops.kv_copy_pages([0], [0], [1]),
                 lambda: ops.token_logprobs(3, pos, 1)):
        with pytest.raises(TypeError, match="tensor"):
            call()


def test_native_module_formats_its_errors():
    """Numbers in a message go through the C++ runtime's streams: they need the runtime that torch uses."""
    with pytest.raises(TypeError, match="takes 9 arguments, got 1"):
        ops._native.paged_flash_decode(1)
    with pytest.raises(ValueError, match="null entry point"):
        ops._native.bind(0, 0, 0, 0, 0, 0)


class LogprobBackend:
    """Logits that peak at the next id, and likelihoods as the engine wants them."""

    def __init__(self, batch):
        self.batch, self.max_seq, self.asked = batch, 32, []

    def _row(self, tok):
        x = torch.zeros(11)
        x[(tok + 1) % 11] = 3.0
        return x

    def prefill(self, slot, prompt):
        return self._row(prompt[-1])

    def step(self, tokens, positions):
        return torch.stack([self._row(t) for t in tokens])

    def logprobs(self, logits, tokens, k):
        self.asked.append((logits.shape[0], list(tokens), k))
        lp = torch.log_softmax(logits, -1)
        return [serve.TokenLogprob(t, float(r[t]), 1, 0.0, tuple((i, float(r[i])) for i in r.topk(k).indices.tolist()))
                for t, r in zip(tokens, lp)]


def test_engine_collects_likelihoods_for_the_requests_that_want_them():
    be = LogprobBackend(3)
    eng = serve.BatchedEngine(be)
    seen = []
    a = eng.submit([1], max_new_tokens=3, logprobs=2, on_token=lambda r, t: seen.append(len(r.token_logprobs)))
    b = eng.submit([5], max_new_tokens=2)
    c = eng.submit([7], max_new_tokens=3, logprobs=0)
    eng.run()
    assert a.tokens == [2, 3, 4] and b.tokens == [6, 7] and c.tokens == [8, 9, 10]
    assert [x.token for x in a.token_logprobs] == a.tokens and seen == [1, 2, 3]
    assert all(len(x.top) == 2 and x.top[0] == (x.token, x.logprob) for x in a.token_logprobs)
    assert b.token_logprobs == [] and [x.top for x in c.token_logprobs] == [(), (), ()]
    assert be.asked == [(1, [2], 2), (1, [8], 0), (2, [3, 9], 2), (2, [4, 10], 2)]
    for bad in (-1, 33):
        with pytest.raises(ValueError):
            eng.submit([1], logprobs=bad)


def test_backend_without_likelihoods_refuses_them():
    class Plain:
        batch, max_seq = 1, 8
    with pytest.raises(ValueError, match="log probabilities"):
        serve.BatchedEngine(Plain()).submit([1], logprobs=1)
