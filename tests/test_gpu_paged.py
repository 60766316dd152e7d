"""GPU: the paged FP8 KV cache (writes, attention, page copies, block table)
against plain 64-bit formulas.

Tolerances, from the arithmetic (u = 2^-24, fp32; results rounded once to
fp16: half a step is 2^-11 relative, 2^-25 below the normal range):
* written q and k: the norm is a sum of 128 squares and a square root, the
  rotation two products, all fp32: (128 + 16) u of |a| + |b| at most, a, b the
  rotated pair, then the rounding.  A stored code must be the code of some
  value that close to the exact one (the codec is monotonic), without norm
  and rotation it is the oracle's encoder bit for bit;
* attention: a score is a sum of 128 exact products in fp32, off by 128 u of
  sum |q k|; weights are e^(score), so off by twice that (numerator and sum),
  plus 2^-21 for the exponential and 2^-21 for carrying a weight as a pair of
  fp16 numbers, plus (64 + n/8) u for sums over n positions on tensor cores;
  all of it times sum p |v|.  A pair ends at 2^-40 of the largest weight (an fp16
  step of 2^-24, halved, of weights carried times 2^15), whatever its own weight
  is: 2^-40 sum |v| / sum e, with sum e >= 1 the weights relative to the largest.
  Then the rounding.  The H32 transform adds 32
  such errors and divides by sqrt(32), with 6 u of its own."""
import numpy as np
import pytest
import torch

import r4q_oracle as O
from test_gpu_gemv import close

pytestmark = pytest.mark.gpu
D, U = 128, 2.0 ** -24
STALE = 0x7F                     # decodes to NaN on the hardware: bytes that must never be used


def dev():
    return torch.device("cuda", torch.cuda.current_device())


def decode_lut():
    return torch.from_numpy(O.fp8_decode(np.arange(256, dtype=np.uint8)).astype(np.float64)).cuda()


def make_paged(lens, Hk, page, seed, scaled=False, spare=3, interleaved=False, std=1.0):
    """Pages in scattered order holding random codes for every position of lens,
    STALE bytes everywhere else.  -> k_pages, v_pages, table, k_scale, v_scale"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = [-(-n // page) for n in lens]
    P = sum(blocks) + spare
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    if interleaved:
        both = torch.full((P, 2, Hk, page, D), STALE, dtype=torch.uint8, device="cuda")
        pages = [both[:, 0], both[:, 1]]
    else:
        pages = [torch.full((P, Hk, page, D), STALE, dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.full((len(lens), max(1, max(blocks)) + 1), P + 7, dtype=torch.int32)   # unused cells: no page at all
    at = 0
    for b, n in enumerate(lens):
        ids = order[at:at + blocks[b]]
        at += blocks[b]
        table[b, :blocks[b]] = torch.tensor(ids, dtype=torch.int32)
        for pg in pages:
            for i, p in enumerate(ids):
                rows = min(page, n - i * page)
                x = torch.randn(Hk, rows, D, generator=g, device="cuda") * (40.0 if scaled else std)
                pg[p, :, :rows] = torch.from_numpy(O.fp8_encode(x.cpu().numpy())).cuda()
    sc = [(0.01 + 0.02 * torch.rand(Hk, generator=g, device="cuda")) if scaled else None for _ in range(2)]
    return pages[0], pages[1], table.cuda(), sc[0], sc[1]


def ref_attention(q, kp, vp, table, lens, ks, vs, fwht):
    """(o, tolerance) in 64 bits, sequence by sequence and head by head."""
    lut, page, Hk = decode_lut(), kp.shape[2], kp.shape[1]
    B, H, _ = q.shape
    Hg = H // Hk
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = table[b, :-(-n // page)].long()
        for h in range(Hk):
            K = lut[kp[ids, h].reshape(-1, D)[:n].long()] * (1 if ks is None else ks[h].double())
            Vv = lut[vp[ids, h].reshape(-1, D)[:n].long()] * (1 if vs is None else vs[h].double())
            qq = q[b, h * Hg:(h + 1) * Hg].double() / np.sqrt(D)
            p = torch.softmax(qq @ K.t(), -1)
            err = 2 * 128 * U * (qq.abs() @ K.abs().t()).amax(-1) + 2.0 ** -20 + (64 + n / 8) * U
            out[b, h * Hg:(h + 1) * Hg] = p @ Vv
            tol[b, h * Hg:(h + 1) * Hg] = err[:, None] * (p @ Vv.abs()) + 2.0 ** -40 * Vv.abs().sum(0)
    if fwht:
        hm = torch.from_numpy(O.hadamard_matrix(32).astype(np.float64)).cuda()
        hm = hm / hm[0].norm()
        mag = out.abs().view(B, H, 4, 32).sum(-1, keepdim=True)
        tol = ((tol.view(B, H, 4, 32).sum(-1, keepdim=True) + 6 * U * mag) / np.sqrt(32)).expand(B, H, 4, 32)
        tol = tol.reshape(B, H, D)
        out = (out.view(B, H, 4, 32) @ hm).reshape(B, H, D)
    return out, tol + out.abs() * 2.0 ** -11 + 2.0 ** -25


def check_attention(o, ref, tol):
    assert torch.isfinite(o).all()
    over = ((o.double() - ref).abs() / tol).max().item()
    assert over <= 1, over


CASES = [  # heads, kv heads, page, lengths, scaled, fwht
    (40, 8, 64, [1], False, False),
    (40, 8, 16, [128], False, True),
    (40, 8, 64, [0, 1, 63, 64, 65, 300], False, True),
    (32, 4, 16, [15, 16, 17, 0, 33, 700], True, False),
    (32, 4, 48, [47, 48, 49, 95, 1000], True, True),
    (8, 8, 32, [31, 32, 33, 0, 0, 257], False, False),
    (16, 1, 128, [5, 1025], True, True),              # 16 heads share one: more than one group of 8
    (12, 1, 16, [77], False, False),                  # a group that 8 does not divide
    (9, 3, 112, [111, 113, 2000], False, True),
    (5, 1, 256, [4000, 3, 255], False, False),
    (2, 2, 1024, [1023, 5000], False, True),
    (40, 8, 64, [9001], True, True),
    (4, 2, 16, [1] * 70 + [0, 400], False, False),    # many short sequences
    (8, 1, 32, [20000, 1, 1], False, False),          # one long among short ones
]


@pytest.mark.parametrize("H,Hk,page,lens,scaled,fwht", CASES)
def test_attention_vs_64_bits(H, Hk, page, lens, scaled, fwht):
    from r4q import ops
    kp, vp, table, ks, vs = make_paged(lens, Hk, page, seed=sum(lens) + H, scaled=scaled)
    q = torch.randn(len(lens), H, D, generator=torch.Generator("cuda").manual_seed(1), device="cuda").half()
    seq = torch.tensor(lens, device="cuda")
    o = ops.paged_flash_decode(q, kp, vp, table, seq, k_scale=ks, v_scale=vs, fwht=fwht)
    check_attention(o, *ref_attention(q, kp, vp, table, lens, ks, vs, fwht))
    assert all(not o[b].any() for b, n in enumerate(lens) if n == 0)
    assert torch.equal(o, ops.paged_flash_decode(q, kp, vp, table, seq, k_scale=ks, v_scale=vs, fwht=fwht))
    ops.check_status()


def test_attention_large_scores_and_spread():
    """Scores of several hundred: one position takes all the weight, and the maximum moves late in the sequence."""
    from r4q import ops
    lens = [1500, 40]
    kp, vp, table, _, _ = make_paged(lens, 2, 32, seed=9, std=6.0)
    q = (torch.randn(2, 8, D, generator=torch.Generator("cuda").manual_seed(2), device="cuda") * 20).half()
    o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor(lens, device="cuda"))
    check_attention(o, *ref_attention(q, kp, vp, table, lens, None, None, False))


def test_attention_small_weights_keep_their_digits():
    """One position takes nearly all the weight and has V = 0: what comes out is the sum of weights around 2^-22."""
    from r4q import ops
    n = 300
    kp, vp, table, _, _ = make_paged([n], 1, 16, seed=15, std=0.3)
    first = table[0, 0].long()
    kp[first, 0, 0], vp[first, 0, 0] = 0, 0
    kp[first, 0, 0, 0] = 0x58                         # 16.0
    q = torch.zeros(1, 8, D, device="cuda").half()
    q[:, :, 0] = 10.75 + 0.01 * torch.arange(8, device="cuda")
    o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor([n], device="cuda"))
    ref, tol = ref_attention(q, kp, vp, table, [n], None, None, False)
    assert ref.abs().max() < 1e-4
    check_attention(o, ref, tol)


def test_attention_scores_of_any_finite_size():
    """All scores alike, at -1e31 and at +1e31: the plain mean of V (a bound that a mask value could be mistaken for)."""
    from r4q import ops
    kp, vp, table, _, _ = make_paged([70], 1, 16, seed=12)
    kp[table[0, :5].long()] = 0x38                    # 1.0
    sc = torch.tensor([1e30], device="cuda")
    ids = table[0, :5].long()
    mean = decode_lut()[vp[ids, 0].reshape(-1, D)[:70].long()]
    for sign in (-1.0, 1.0):
        q = torch.full((1, 8, D), sign, device="cuda").half()
        o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor([70], device="cuda"), k_scale=sc)
        tol = mean.abs().mean(0) * (2.0 ** -20 + 80 * U) + mean.mean(0).abs() * 2.0 ** -11 + 2.0 ** -25
        assert ((o[0].double() - mean.mean(0)).abs() <= tol).all()


@pytest.mark.parametrize("top", [t << e for e in range(21, 27) for t in (9, 13, 15)])
def test_attention_scores_whose_steps_exceed_one(top):
    """Half the scores at about `top` (1.9e7 .. 1.0e9, where fp32 steps are 2 .. 64), half at 1 / 8 of it: the mean of V
    over the first half, which takes every position's weight to be equal and no larger than fp16 holds."""
    from r4q import ops
    n = 96
    kp, vp, table, _, _ = make_paged([n], 1, 16, seed=13)
    ids = table[0, :n // 16].long()
    kp[ids] = 0x28                                    # 0.25 = 2 / 8
    kp[ids[::2]] = 0x40                               # 2.0
    mean = decode_lut()[vp[ids[::2], 0].reshape(-1, D).long()]
    q = (1 + torch.arange(8, device="cuda") / 64)[None, :, None].expand(1, 8, D).half()
    scale = torch.tensor([top / (2 * D / D ** 0.5 * 1.4426950408889634)], device="cuda")
    o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor([n], device="cuda"), k_scale=scale)
    tol = mean.abs().mean(0) * (2.0 ** -20 + (64 + n / 8) * U) + mean.mean(0).abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((o[0].double() - mean.mean(0)).abs() <= tol).all()


def test_attention_views_strides_and_shared_pages():
    """q out of a wider row, K and V interleaved in one pool, a table with wider rows and more of them than the
    batch, an output with its own stride; two sequences on the same pages give the same result."""
    from r4q import ops
    lens = [130, 45, 130]
    kp, vp, table, _, _ = make_paged(lens, 2, 32, seed=4, interleaved=True)
    table[2] = table[0]
    qkv = torch.randn(3, (6 + 4) * D, generator=torch.Generator("cuda").manual_seed(3), device="cuda").half()
    qkv[2] = qkv[0]
    q = qkv[:, :6 * D].view(3, 6, D)
    wide = torch.full((5, table.shape[1] + 3), 1 << 20, dtype=torch.int32, device="cuda")
    wide[:3, :table.shape[1]] = table
    buf = torch.full((3, 9, D), 7.0, dtype=torch.float16, device="cuda")
    o = ops.paged_flash_decode(q, kp, vp, wide[:, :table.shape[1]], torch.tensor(lens, device="cuda"), out=buf[:, 2:8])
    ref, tol = ref_attention(q, kp, vp, table, lens, None, None, False)
    check_attention(o, ref, tol)
    assert torch.equal(o[0], o[2]) and (buf[:, :2] == 7).all() and (buf[:, 8:] == 7).all()
    # heads apart: copied by the wrapper
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(o, ops.paged_flash_decode(qt, kp, vp, table, torch.tensor(lens, device="cuda")))
    ops.check_status()


def test_attention_agrees_with_the_contiguous_cache():
    """Same bytes, same arithmetic up to the order of sums: twice the bound of each."""
    from r4q import ops
    n, H, Hk, page = 777, 40, 8, 64
    kp, vp, table, _, _ = make_paged([n], Hk, page, seed=6)
    q = torch.randn(1, H, D, generator=torch.Generator("cuda").manual_seed(4), device="cuda").half()
    o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor([n], device="cuda"), fwht=True)
    ids = table[0, :-(-n // page)].long()
    kc, vc = (p[ids].permute(1, 0, 2, 3).reshape(1, Hk, -1, D)[:, :, :n].contiguous() for p in (kp, vp))
    c = ops.flash_decode(q, kc, vc, n, fwht=True)
    close(o.cpu().numpy(), c.float().cpu().numpy())


def test_attention_streams_and_graphs_share_nothing():
    """Two captured graphs and two streams at once, each with its own lengths; replays read the lengths, the table
    and q as they are at that time."""
    from r4q import ops
    lens = [[3000, 10, 200], [700, 1300, 1]]
    sets = [make_paged(n, 4, 32, seed=20 + i) for i, n in enumerate(lens)]
    qs = [torch.randn(3, 16, D, generator=torch.Generator("cuda").manual_seed(i), device="cuda").half() for i in (5, 6)]
    seqs = [torch.tensor(n, device="cuda") for n in lens]
    refs = [ref_attention(qs[i], *sets[i][:3], lens[i], None, None, False) for i in (0, 1)]
    ops.paged_flash_decode(qs[0], *sets[0][:3], seqs[0])
    torch.cuda.synchronize()
    cap = torch.cuda.Stream()
    graphs, outs = [], []
    for i in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            outs.append(ops.paged_flash_decode(qs[i], *sets[i][:3], seqs[i]))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
                eager[1 - i].append(ops.paged_flash_decode(qs[1 - i], *sets[1 - i][:3], seqs[1 - i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        check_attention(outs[i], *refs[i])
        assert all(torch.equal(e, eager[i][0]) for e in eager[i]) and torch.equal(eager[i][0], outs[i])
    seqs[0].copy_(torch.tensor([0, 10, 100]))
    graphs[0].replay()
    torch.cuda.synchronize()
    check_attention(outs[0], *ref_attention(qs[0], *sets[0][:3], [0, 10, 100], None, None, False))
    ops.check_status()


def test_first_call_may_be_captured(tmp_path):
    """In a fresh process, all operators for the first time under capture: nothing has to be warmed up."""
    import subprocess
    import sys
    from conftest import PKG
    code = f"""
import sys; sys.path.insert(0, {str(PKG)!r})
import torch
from r4q import ops
z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype, device="cuda")
pool, table, k = z(1, 2, 64, 2, 16, 128), torch.arange(60, dtype=torch.int32, device="cuda").view(2, 30), z(2, 2, 128, dtype=torch.half)
pos, x = torch.tensor([0, 400], device="cuda"), torch.randn(3, 9000, device="cuda").half()
k += 1
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.paged_kv_write(k, k, pool[0, 0], pool[0, 1], table, pos)
    o = ops.paged_flash_decode(k, pool[0, 0], pool[0, 1], table, pos + 1)
    ops.kv_copy_pages(pool, [0], [63])
    ops.kv_table_set(table, [1], [29], [63])
    r = ops.token_logprobs(x, x.argmax(-1), 4)
g.replay()
torch.cuda.synchronize()
ops.check_status()
assert (o[0] == 1).all() and torch.isfinite(o).all() and (r.rank == 1).all()
assert torch.equal(pool[:, :, 63], pool[:, :, 0]) and pool[0, 0, 0].any() and table[1, 29] == 63
print("captured")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_attention_reports_bad_pages_and_lengths():
    from r4q import lib as L, ops
    kp, vp, table, _, _ = make_paged([100, 100], 2, 16, seed=8)
    q = torch.randn(2, 4, D, device="cuda").half()
    seq = torch.tensor([100, 100], device="cuda")
    good = ops.paged_flash_decode(q, kp, vp, table, seq)
    ops.check_status()
    for bad in (-1, kp.shape[0], 1 << 30, -(1 << 31)):
        t = table.clone()
        t[1, 3] = bad
        o = ops.paged_flash_decode(q, kp, vp, t, seq)
        with pytest.raises(L.R4QError) as e:
            ops.check_status()
        assert e.value.code == -6
        assert torch.equal(o[0], good[0]) and torch.isfinite(o).all()
    for n in (table.shape[1] * 16 + 1, 1 << 40, -1):
        o = ops.paged_flash_decode(q, kp, vp, table, torch.tensor([100, n], device="cuda"))
        with pytest.raises(L.R4QError):
            ops.check_status()
        assert torch.equal(o[0], good[0])
    ops.check_status()                                # cleared


# ------------------------------------------------------------------- writes ---
def ref_head(x, w, cos, sin, norm, rope, eps=1e-6):
    """(value, tolerance) of the normalised and rotated heads [M, h, 128] in 64 bits."""
    x = x.double()
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    tol = x.abs() if norm else x.abs() * 0
    if rope:
        a, b, c, s = x[..., :64], x[..., 64:], cos.double()[:, None, :64], sin.double()[:, None, :64]
        x = torch.cat([a * c - b * s, b * c + a * s], -1)
        tol = (a.abs() + b.abs()).repeat(1, 1, 2)
    return x, tol * 144 * U


def check_codes(codes, x, tol, scale):
    """Each code lies between the codes of x - tol and x + tol."""
    s = 1 if scale is None else scale.double()[None, :, None]
    lut = O.fp8_decode(np.arange(256, dtype=np.uint8)).astype(np.float64)
    got = lut[codes.cpu().numpy()]
    lo, hi = (lut[O.fp8_encode((y / s * (1 + sgn * 4 * U * torch.sign(y))).cpu().numpy().astype(np.float32))]
              for y, sgn in ((x - tol, -1), (x + tol, 1)))
    assert (got >= lo).all() and (got <= hi).all()


WRITES = [  # heads of q, kv heads, page, tokens, norm, rope, scaled
    (40, 8, 64, 1, True, True, False),
    (40, 8, 16, 37, True, True, True),
    (0, 4, 48, 100, False, False, True),
    (0, 8, 32, 129, False, False, False),
    (32, 4, 16, 513, True, True, False),
    (3, 1, 128, 50, True, False, False),
    (5, 5, 16, 70, False, True, True),
    (0, 3, 16, 33, True, True, False),
]


@pytest.mark.parametrize("H,Hk,page,M,norm,rope,scaled", WRITES)
def test_write_vs_64_bits(H, Hk, page, M, norm, rope, scaled):
    """Tokens of five ragged sequences in mixed order, padding among them, into scattered pages."""
    from r4q import ops
    rng = np.random.default_rng(M + H)
    S, nb = 5, 2 * M // page + 3
    P = S * nb + 2
    table = torch.from_numpy(rng.permutation(P)[:S * nb].reshape(S, nb).astype(np.int32)).cuda()
    slots = rng.permutation(S * nb * page)[:M]
    rows = torch.from_numpy((slots // (nb * page)).astype(np.int32)).cuda()
    pos = torch.from_numpy((slots % (nb * page)).astype(np.int64)).cuda()
    pos[rng.random(M) < 0.15] = -1
    if M == 1:
        pos[0] = nb * page - 1
    g = torch.Generator("cuda").manual_seed(M)
    qkv = torch.randn(M, (H + 2 * Hk) * D + 8, generator=g, device="cuda").half() * 3
    q = qkv[:, :H * D].view(M, H, D) if H else None
    k, v = (qkv[:, o * D:(o + Hk) * D].view(M, Hk, D) for o in (H, H + Hk))
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).half() for _ in range(2)]
    ang = torch.randn(nb * page, 64, generator=g, device="cuda") * 9
    cos, sin = ang.cos().half(), ang.sin().half()
    sc = [0.3 * torch.rand(Hk, generator=g, device="cuda") + 0.01 if scaled else None for _ in range(2)]
    kp, vp = (torch.full((P, Hk, page, D), STALE, dtype=torch.uint8, device="cuda") for _ in range(2))
    want_k, want_v = kp.clone(), vp.clone()
    kout = torch.full((M, Hk, D), 7.0, dtype=torch.float16, device="cuda")
    qout = torch.full((M, H, D), 7.0, dtype=torch.float16, device="cuda") if H else None
    kw = dict(q_w=w[0] if H else None, k_w=w[1]) if norm else {}
    kw.update(dict(cos=cos, sin=sin) if rope else {})
    r = ops.paged_kv_write(k, v, kp, vp, table, pos, rows=rows, q=q, q_out=qout, k_out=kout, k_scale=sc[0],
                           v_scale=sc[1], **kw)
    live = pos >= 0
    at = pos.clamp(min=0)
    page_of = table[rows.long(), at // page].long()
    kr, kt = ref_head(k, w[1], cos[at], sin[at], norm, rope)
    half = lambda y: y.abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((kout.double() - kr).abs() <= kt + half(kr))[live].all() and (kout[~live] == 7).all()
    if H:
        qr, qt = ref_head(q, w[0], cos[at], sin[at], norm, rope)
        assert r is qout and ((r.double() - qr).abs() <= qt + half(qr))[live].all() and (r[~live] == 7).all()
    got_k, got_v = kp[page_of, :, at % page][live], vp[page_of, :, at % page][live]
    enc = lambda y, s: torch.from_numpy(O.fp8_encode(
        (y.float() if s is None else y.float() / s[None, :, None]).cpu().numpy())).cuda()
    assert torch.equal(got_v, enc(v, sc[1])[live])
    if norm or rope:
        check_codes(got_k, kr[live], kt[live], sc[0])
    else:
        assert torch.equal(got_k, enc(k, sc[0])[live])
    for pool, want, got in ((kp, want_k, got_k), (vp, want_v, got_v)):     # nothing else was written
        want[page_of[live], :, at[live] % page] = got
        assert torch.equal(pool, want)
    ops.check_status()


def test_write_full_range_codec():
    """Every fp16 value, divided by scales among them: three mantissa bits, ties away from zero, 0 below 2^-6 (what
    rounds up to it excepted), at most 448; and the reader decodes it.  Without full_range: the oracle's encoder."""
    from r4q import ops
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x)][:63488].cuda().view(-1, 1, D)
    M, page = x.shape[0], 16
    table = torch.arange(M // page, dtype=torch.int32, device="cuda")[None]
    kp, vp = (torch.zeros(M // page, 1, page, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.tensor([0.37], device="cuda")
    args = (x, x, kp, vp, table, torch.arange(M, device="cuda"))
    rows = torch.zeros(M, dtype=torch.int32, device="cuda")
    ops.paged_kv_write(*args, rows=rows, v_scale=sc, full_range=True)
    lut = decode_lut()
    for pool, y in ((kp, x.float()), (vp, x.float() / sc)):
        a = y.double().abs().clamp(max=448.0)
        step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -30))) - 3)
        want = torch.floor(a / step + 0.5) * step
        want = torch.where(want < 2.0 ** -6, 0 * want, want) * torch.sign(y.double())
        got = lut[pool.view(M, 1, D).long()]
        assert torch.equal(got, want) and got.abs().max() == 448 and (got.abs() == 320).any()
    ops.paged_kv_write(*args, rows=rows, v_scale=sc)
    for pool, y in ((kp, x.float()), (vp, x.float() / sc)):
        assert torch.equal(pool.view(M, 1, D).cpu(), torch.from_numpy(O.fp8_encode(y.cpu().numpy())))
    o = ops.paged_flash_decode(torch.zeros(1, 1, D, device="cuda").half(), kp, vp, table,
                               torch.tensor([1], device="cuda"))
    assert torch.isfinite(o).all()


def test_write_default_rows_in_place_and_captured():
    """A decode step's form: token m of sequence m, q rotated in place; captured and replayed at later positions."""
    from r4q import ops
    g = torch.Generator("cuda").manual_seed(3)
    H, Hk, page, B = 4, 2, 16, 3
    qkv = torch.randn(B, (H + 2 * Hk) * D, generator=g, device="cuda").half()
    src = qkv.clone()
    q, k, v = (qkv[:, o * D:(o + n) * D].view(B, n, D) for o, n in ((0, H), (H, Hk), (H + Hk, Hk)))
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).half()
    ang = torch.randn(64, 64, generator=g, device="cuda")
    cos, sin = ang.cos().half(), ang.sin().half()
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(B, 4)
    kp, vp = (torch.zeros(12, Hk, page, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    pos = torch.zeros(B, dtype=torch.int64, device="cuda")

    def step():
        qkv.copy_(src)
        return ops.paged_kv_write(k, v, kp, vp, table, pos, q=q, q_w=w, k_w=w, cos=cos, sin=sin, q_out=q)
    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    assert out is q
    for ps in ([5, 17, 63], [6, -1, 31]):
        kp.zero_()
        pos.copy_(torch.tensor(ps))
        gr.replay()
        torch.cuda.synchronize()
        for b, p in enumerate(ps):
            if p < 0:
                assert torch.equal(qkv[b], src[b])
                continue
            ref, tol = ref_head(src[b:b + 1, :H * D].view(1, H, D), w, cos[p:p + 1], sin[p:p + 1], True, True)
            assert ((q[b].double() - ref[0]).abs() <= tol[0] + ref[0].abs() * 2.0 ** -11 + 2.0 ** -25).all()
            assert kp[table[b, p // page].item(), :, p % page].any()
        assert int(kp.any(-1).sum()) == Hk * sum(p >= 0 for p in ps)
    ops.check_status()


def test_write_reports_what_is_out_of_range():
    from r4q import lib as L, ops
    k = torch.randn(2, 2, D, device="cuda").half()
    kp, vp = (torch.zeros(4, 2, 16, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.tensor([[0, 1], [2, 4], [-1, 3]], dtype=torch.int32, device="cuda")
    cos = torch.ones(20, 64, dtype=torch.float16, device="cuda")
    def call(rows, pos, **kw):
        kp.zero_(), vp.zero_()
        ops.paged_kv_write(k, k, kp, vp, table, torch.tensor(pos, device="cuda"),
                           rows=torch.tensor(rows, dtype=torch.int32, device="cuda"), **kw)
    for rows, pos, kw in (([0, 3], [1, 1], {}), ([0, -1], [1, 1], {}), ([0, 0], [1, 32], {}), ([0, 1], [1, 16], {}),
                          ([0, 2], [1, 0], {}), ([0, 0], [1, 1 << 40], {}), ([0, 0], [1, 21], dict(cos=cos, sin=cos))):
        call(rows, pos, **kw)
        with pytest.raises(L.R4QError) as e:
            ops.check_status()
        assert e.value.code == -6
        assert kp[0, :, 1].any() and int(kp.any(-1).sum()) == 2 and int(vp.any(-1).sum()) == 2
    call([0, 1], [1, 15])
    ops.check_status()


# -------------------------------------------------------------- page copies ---
@pytest.mark.parametrize("lead,P,Hk,page,n", [((), 5, 1, 16, 1), ((3, 2), 7, 2, 16, 3), ((2,), 3000, 1, 16, 1400),
                                              ((40, 2), 9, 8, 64, 2), ((1, 2), 4, 3, 48, 2)])
def test_copy_pages_and_table(lead, P, Hk, page, n):
    from r4q import ops
    g = torch.Generator("cuda").manual_seed(P)
    pool = torch.randint(0, 256, (*lead, P, Hk, page, D), generator=g, device="cuda", dtype=torch.uint8)
    rng = np.random.default_rng(n)
    ids = rng.permutation(P)
    dst = ids[:n].tolist()
    src = rng.choice(ids[n:], size=n).tolist()          # one page may go to several places
    want = pool.clone()
    want[..., torch.tensor(dst, device="cuda"), :, :, :] = pool[..., torch.tensor(src, device="cuda"), :, :, :]
    ops.kv_copy_pages(pool, src, torch.tensor(dst))
    assert torch.equal(pool, want)
    table = torch.randint(0, 99, (60, 70), generator=g, device="cuda", dtype=torch.int32)
    cells = rng.permutation(60 * 50)[:n]
    tw = table.clone()
    tw[torch.from_numpy(cells // 50), torch.from_numpy(cells % 50)] = torch.tensor(dst, dtype=torch.int32, device="cuda")
    ops.kv_table_set(table[:, :50], (cells // 50).tolist(), torch.from_numpy(cells % 50), dst)
    assert torch.equal(table, tw)


def test_wrapper_refusals_on_device_tensors():
    from r4q import ops
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype, device="cuda")
    pg, t, k = z(4, 2, 16, D), z(3, 4, dtype=torch.int32), z(3, 2, D, dtype=torch.float16)
    pos = z(3, dtype=torch.int64)
    bad = [
        lambda: ops.paged_flash_decode(k.float(), pg, pg, t, pos),
        lambda: ops.paged_flash_decode(k, pg.to(torch.int8), pg, t, pos),
        lambda: ops.paged_flash_decode(k, pg, z(4, 2, 32, D), t, pos),
        lambda: ops.paged_flash_decode(k, pg.transpose(1, 2).contiguous().transpose(1, 2), pg, t, pos),
        lambda: ops.paged_flash_decode(k, pg, pg, t.long(), pos),
        lambda: ops.paged_flash_decode(k, pg, pg, t, pos.int()),
        lambda: ops.paged_flash_decode(k, pg, pg, t, pos[:2]),
        lambda: ops.paged_flash_decode(k, pg, pg, t, pos, k_scale=z(3, 2, dtype=torch.float32)),
        lambda: ops.paged_flash_decode(k, pg, pg, t, pos, out=z(3, 2, 2 * D, dtype=torch.float16)[..., ::2]),
        lambda: ops.paged_kv_write(k, k[:2], pg, pg, t, pos),
        lambda: ops.paged_kv_write(k, k, pg, pg, t, pos, rows=pos),
        lambda: ops.paged_kv_write(k, k, pg, pg, t, pos, q_out=k),
        lambda: ops.paged_kv_write(k, k, pg, pg, t, pos, q=k, k_w=z(D, dtype=torch.float16)),
        lambda: ops.paged_kv_write(k, k, pg, pg, t, pos, cos=z(9, 64, dtype=torch.float16)),
        lambda: ops.kv_copy_pages(pg[:, :1], [0], [1]),
        lambda: ops.kv_copy_pages(pg, pos, [1]),
        lambda: ops.kv_table_set(t.t(), [0], [0], [0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((TypeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")


def test_pools_beyond_32_bit_offsets():
    """5 GB each of K and V in one interleaved pool, the used pages at both ends: write, attention, copy."""
    from r4q import ops
    Hk, page, P = 8, 64, 80000
    pool = torch.zeros(2, P, Hk, page, D, dtype=torch.uint8, device="cuda")
    g = torch.Generator("cuda").manual_seed(3)
    n = 150
    table = torch.tensor([[P - 1, 0, P - 7], [1, P // 2, 2]], dtype=torch.int32, device="cuda")
    lens = [n, 70]
    k, v = (torch.randn(sum(lens), Hk, D, generator=g, device="cuda").half() for _ in range(2))
    pos = torch.cat([torch.arange(m) for m in lens]).cuda()
    rows = torch.cat([torch.full((m,), i) for i, m in enumerate(lens)]).int().cuda()
    ops.paged_kv_write(k, v, pool[0], pool[1], table, pos, rows=rows)
    q = torch.randn(2, 16, D, generator=g, device="cuda").half()
    seq = torch.tensor(lens, device="cuda")
    o = ops.paged_flash_decode(q, pool[0], pool[1], table, seq)
    check_attention(o, *ref_attention(q, pool[0], pool[1], table, lens, None, None, False))
    ops.kv_copy_pages(pool, [P - 1, P - 7], [P - 2, 3])
    ops.kv_table_set(table, [0, 0], [0, 2], [P - 2, 3])
    assert torch.equal(ops.paged_flash_decode(q, pool[0], pool[1], table, seq), o)
    ops.check_status()


# ------------------------------------------------------------- used together ---
def test_cache_life_prefix_forks_copies_compaction():
    """Sequences prefilled, forked, extended (a shared page is copied before it is written), freed and compacted;
    after every step the attention of every sequence equals 64-bit attention over the tokens it was given."""
    from r4q import ops, paged
    H, Hk, page, layers, S = 8, 2, 16, 2, 4
    c = paged.PagedKVCache(layers, 24, Hk, page, S, 10, dev())
    g = torch.Generator("cuda").manual_seed(11)
    c.pool.fill_(STALE)
    hist = [[torch.zeros(2, 0, Hk, D, dtype=torch.uint8, device="cuda") for _ in range(S)] for _ in range(layers)]

    def add(counts):
        plan = c.extend(counts)
        for li in range(layers):
            ks, vs, rows, pos = [], [], [], []
            for s, n in counts.items():
                kv = torch.randn(2, n, Hk, D, generator=g, device="cuda").half()
                codes = torch.from_numpy(O.fp8_encode(kv.float().cpu().numpy())).cuda()
                start = hist[li][s].shape[1]
                hist[li][s] = torch.cat([hist[li][s], codes], 1)
                ks.append(kv[0]), vs.append(kv[1])
                rows += [s] * n
                pos += list(range(start, start + n))
            ops.paged_kv_write(torch.cat(ks), torch.cat(vs), *c.pages(li), c.table, torch.tensor(pos, device="cuda"),
                               rows=torch.tensor(rows, dtype=torch.int32, device="cuda"), **c.scales(li))
        return plan

    def check():
        lens = list(c.lengths)
        q = torch.randn(S, H, D, generator=g, device="cuda").half()
        for li in range(layers):
            o = ops.paged_flash_decode(q, *c.pages(li), c.table, torch.tensor(lens, device="cuda"))
            flat = torch.cat([hist[li][s] for s in range(S)], 1)      # each history as one page of its own
            n = max(16, -(-max(lens) // 16) * 16)
            pools = torch.zeros(2, S, Hk, n, D, dtype=torch.uint8, device="cuda")
            for s in range(S):
                pools[:, s, :, :lens[s]] = hist[li][s].transpose(1, 2)
            assert flat.shape[1] == sum(lens)
            own = torch.arange(S, dtype=torch.int32, device="cuda")[:, None]
            check_attention(o, *ref_attention(q, pools[0], pools[1], own, lens, None, None, False))
        ops.check_status()

    add({0: 37, 1: 20})
    check()
    c.fork(0, 2)
    c.fork(0, 3, 20)
    for li in range(layers):
        hist[li][2], hist[li][3] = hist[li][0], hist[li][0][:, :20]
    check()
    plan = add({0: 3, 2: 30, 3: 1})
    assert len(plan.src) == 2 and c.free_count < 24
    check()
    c.free(0)
    for li in range(layers):
        hist[li][0] = hist[li][0][:, :0]
    check()
    assert c.compact().src
    check()
    add({0: 17, 1: 1, 2: 1, 3: 1})
    check()


CFG = dict(num_layers=2, hidden=256, num_heads=4, num_kv_heads=2, head_dim=128, experts=16, topk=4, expert_inter=128,
           vocab=512, rms_eps=1e-6, rope_theta=1e6)


def test_moe_decoder_on_pages_agrees_with_the_contiguous_cache():
    """One layer, so that both decoders see the same qkv in every step: the paged cache then holds the contiguous
    one's bytes bit for bit, and each step's logits lie within the decode step's tolerance (2e-3) of the exact ones
    for that cache, so within twice that of each other."""
    from r4q import moe, paged
    B, T = 2, 37
    cfg = dict(CFG, num_layers=1)
    m = moe.build_moe_model(cfg, dev(), seed=3, max_seq=64, batch=B)
    tok = torch.randint(0, CFG['vocab'], (T, B), generator=torch.Generator().manual_seed(1)).cuda()
    flat = moe.MoEDecoder(m, cfg, batch=B)
    pages = paged.PagedKVCache(1, 14, 2, 16, B, 4, dev())
    dec = moe.MoEDecoder(m, cfg, batch=B, pages=pages)
    for t in range(T):
        a = flat.step(m['embed'][tok[t]], t).float().cpu().numpy()
        pages.extend({0: 1, 1: 1})
        b = dec.step(m['embed'][tok[t]], t)
        close(b.float().cpu().numpy(), a, 2 * 2e-3)
    for pool, flat_cache in zip(pages.pages(0), (m['k_caches'][0], m['v_caches'][0])):
        for b in range(B):
            got = pool[pages.table[b, :3].long()].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :T]
            assert torch.equal(got, flat_cache[b, :, :T])


def test_moe_decoder_on_pages_forks_idles_and_compacts():
    """Graph replay equals the eager step bit for bit, a fork continues its parent's sequence beside it with equal
    logits, an idle row writes nothing, and the sampled tokens' likelihoods match the logits."""
    from r4q import moe, ops, paged
    B, T = 3, 21
    m = moe.build_moe_model(CFG, dev(), seed=3, max_seq=64, batch=B)
    tok = torch.randint(0, CFG['vocab'], (T, B), generator=torch.Generator().manual_seed(1)).cuda()
    tok[:, 2] = tok[:, 0]
    pages = paged.PagedKVCache(2, 14, 2, 16, B, 4, dev())
    dec = moe.MoEDecoder(m, CFG, batch=B, pages=pages)
    for t in range(T):
        if t < 18:                                    # row 2 forks row 0 at 18
            pages.extend({0: 1, 1: 1})
            b = dec.step(m['embed'][tok[t]], [t, t, -1]).clone()
            assert pages.pool.any(-1).sum() <= 2 * 2 * 2 * 2 * (t + 1)     # layers, K/V, kv heads, two sequences
        else:
            if t == 18:
                pages.fork(0, 2)
            pages.extend({0: 1, 1: 1, 2: 1})
            b = dec.step(m['embed'][tok[t]], t).clone()
            assert torch.equal(b[0], b[2])
    eager = dec.step(m['embed'][tok[T - 1]], torch.tensor([T - 1] * B), use_graph=False)
    assert torch.equal(eager, b)
    r = ops.token_logprobs(b, b.argmax(-1), 3)
    ref = torch.log_softmax(b.double(), -1)
    assert (r.rank == 1).all() and torch.equal(r.top_ids[:, 0], b.argmax(-1))
    assert (r.logprob.double() - ref.max(-1).values).abs().max() < 1e-5
    pages.free(1)
    pages.compact()
    pages.extend({0: 1, 2: 1})
    c = dec.step(m['embed'][tok[0]], [T, -1, T])
    assert torch.equal(c[0], c[2])
    with pytest.raises(ValueError):
        dec.step(m['embed'][tok[0]], [T + 1, -1, T])
    ops.check_status()


def test_moe_decoder_refuses_pages_that_another_sequence_shares():
    """A fork without an extend: a step at a position on a shared page would change what the other sequence reads."""
    from r4q import moe, paged
    m = moe.build_moe_model(CFG, dev(), seed=3, max_seq=64, batch=2)
    pages = paged.PagedKVCache(2, 8, 2, 16, 2, 4, dev())
    dec = moe.MoEDecoder(m, CFG, batch=2, pages=pages)
    x = m['embed'][:2].clone()
    pages.extend({0: 1})
    dec.step(x, [0, -1])
    pages.fork(0, 1)
    before = pages.pool.clone()
    for pos in ([0, -1], [-1, 0], [0, 0]):
        with pytest.raises(ValueError):
            dec.step(x, pos)
    assert torch.equal(pages.pool, before)
    pages.extend({1: 1})
    dec.step(x, [-1, 1])
    dec.step(x, [0, 1])


def test_prefill_into_pages_then_decode_attention():
    """prefill_logits into pages: the logits of a prefill into the contiguous cache (5e-3, the prefill's tolerance),
    and cache codes that differ by a step at most: the paged write encodes K unrounded, the other one from fp16."""
    from r4q import paged, prefill as P, synth
    cfg = dict(num_layers=2, hidden=512, intermediate=1024, num_heads=4, num_kv_heads=2, head_dim=128, vocab=1008,
               rms_eps=1e-6, rope_theta=1e6)
    m = synth.build_decode_model(cfg, dev(), seed=7, max_seq=64, batch=1)
    ids = torch.randint(0, 1008, (45,), generator=torch.Generator().manual_seed(2)).cuda()
    args = (m['embed'][ids], m['qkv_w'], m['qkv_s'], m['o_w'], m['o_s'], m['gu_w'], m['gu_s'], m['down_w'],
            m['down_s'], m['in_norm_w'], m['post_norm_w'], m['q_norm_w'], m['k_norm_w'], m['rope_cos'], m['rope_sin'],
            4, 2, 128, 512, 1024, 1e-6, m['final_norm_w'], m['lm_w'], m['lm_s'], 1008)
    a = P.prefill_logits(*args, k_caches=m['k_caches'], v_caches=m['v_caches'], last_only=True)
    pages = paged.PagedKVCache(2, 8, 2, 16, 3, 4, dev())
    with pytest.raises(ValueError):
        P.prefill_logits(*args, pages=pages, batch_row=1)
    pages.extend({1: 45})
    pages.fork(1, 2, 10)
    with pytest.raises(ValueError, match="shares"):
        P.prefill_logits(*args, pages=pages, batch_row=1)
    pages.free(2)
    b = P.prefill_logits(*args, pages=pages, batch_row=1, last_only=True)
    close(b.float().cpu().numpy(), a.float().cpu().numpy(), 5e-3)
    lut = decode_lut()
    for li, (kc, vc) in enumerate(zip(m['k_caches'][:1], m['v_caches'][:1])):     # layer 0: the same inputs
        kp, vp = (p[pages.table[1, :3].long()].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :45] for p in pages.pages(li))
        assert torch.equal(vp, vc[0, :, :45])
        x, y = lut[kp.long()], lut[kc[0, :, :45].long()]
        assert ((x - y).abs() <= torch.maximum(x.abs(), y.abs()) / 8 + 2.0 ** -6).all()
