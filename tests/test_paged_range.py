"""The page write's codec by default: E4M3's whole range, 448 at most.  The
cache codec of the contiguous kernels (448 from 248 on) is asked for."""
import numpy as np
import pytest
import torch

import r4q_oracle as O
from r4q import ops, paged

D = 128


def test_caches_keep_the_whole_range_unless_told_otherwise():
    c = paged.PagedKVCache(1, 2, 1, 16, 1, 2, "cpu", k_scales=[torch.ones(1)], v_scales=[torch.ones(1)])
    assert c.codec(0)["full_range"] is True
    assert paged.PagedKVCache(1, 2, 1, 16, 1, 2, "cpu", full_range=False).codec(0)["full_range"] is False


def whole_range(y):
    """The value that E4M3 holds for y: three mantissa bits, ties away from zero, 0 below 2^-6, 448 at most."""
    a = y.double().abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -30))) - 3)
    r = torch.floor(a / step + 0.5) * step
    return torch.where(r < 2.0 ** -6, 0 * r, r).clamp(max=448.0) * torch.sign(y.double())


@pytest.mark.gpu
@pytest.mark.parametrize("scaled", [False, True])
def test_default_write_keeps_256_to_448_apart(scaled):
    """Values over the whole range, from 2^-8 to 600 times the scale, written by a call that says nothing of the codec:
    the decoded code is the nearest one (fp16 values and fp32 quotients, so every step is exact or as the formula's)."""
    Hk, M, page = 3, 256, 16
    g = torch.Generator("cuda").manual_seed(5)
    scale = 0.008 + 0.004 * torch.rand(Hk, generator=g, device="cuda") if scaled else torch.ones(Hk, device="cuda")
    size = torch.exp2(torch.rand(2, M, Hk, D, generator=g, device="cuda") * 17.2 - 8)
    x = (size * torch.randn(size.shape, generator=g, device="cuda").sign() * scale[:, None]).half()
    pool = torch.zeros(2, M // page, Hk, page, D, dtype=torch.uint8, device="cuda")
    table = torch.arange(M // page, dtype=torch.int32, device="cuda")[None]
    args = (x[0], x[1], pool[0], pool[1], table, torch.arange(M, device="cuda"))
    kw = dict(rows=torch.zeros(M, dtype=torch.int32, device="cuda"))
    if scaled:
        kw.update(k_scale=scale, v_scale=scale)
    ops.paged_kv_write(*args, **kw)
    y = x.float() / scale[:, None]
    lut = torch.from_numpy(O.fp8_decode(np.arange(256, dtype=np.uint8)).astype(np.float64)).cuda()
    read = lambda: pool.permute(0, 1, 3, 2, 4).reshape(2, M, Hk, D)
    got = lut[read().long()]
    assert torch.equal(got, whole_range(y))
    assert all((got.abs() == v).any() for v in (256, 288, 320, 352, 384, 416, 448))
    ops.paged_kv_write(*args, full_range=False, **kw)
    assert torch.equal(read().cpu(), torch.from_numpy(O.fp8_encode(y.cpu().numpy())))
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("H,Hk,page,M,norm,rope", [(40, 8, 16, 37, True, True), (0, 4, 48, 100, False, False),
                                                   (5, 5, 16, 70, False, True), (3, 1, 32, 9, True, False)])
def test_scaled_writes_vs_64_bits(H, Hk, page, M, norm, rope, full):
    """Normalised and rotated heads over scales that leave a good part of the values beyond 248: each code lies between
    those of the exact value less and plus its error (test_gpu_paged's bound; both codecs are monotonic)."""
    from test_gpu_paged import U, ref_head
    g = torch.Generator("cuda").manual_seed(M)
    S, nb = 2, M // page + 1
    table = torch.randperm(S * nb, generator=torch.Generator().manual_seed(M)).int().view(S, nb).cuda()
    rows = (torch.arange(M, device="cuda") % S).int()
    pos = torch.arange(M, device="cuda") // S
    k, v = (3 * torch.randn(2, M, Hk, D, generator=g, device="cuda")).half()
    q = torch.randn(M, H, D, generator=g, device="cuda").half() if H else None
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).half() for _ in range(2)]
    ang = torch.randn(nb * page, 64, generator=g, device="cuda") * 9
    cos, sin = ang.cos().half(), ang.sin().half()
    sc = [0.005 + 0.02 * torch.rand(Hk, generator=g, device="cuda") for _ in range(2)]
    kp, vp = (torch.zeros(S * nb, Hk, page, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    kw = dict(q_w=w[0] if H else None, k_w=w[1]) if norm else {}
    kw.update(dict(cos=cos, sin=sin) if rope else {}, **({} if full else dict(full_range=False)))
    ops.paged_kv_write(k, v, kp, vp, table, pos, rows=rows, q=q, k_scale=sc[0], v_scale=sc[1], **kw)
    at = table[rows.long(), pos // page].long(), slice(None), pos % page
    lut = torch.from_numpy(O.fp8_decode(np.arange(256, dtype=np.uint8)).astype(np.float64)).cuda()
    held = whole_range if full else lambda y: lut[torch.from_numpy(O.fp8_encode(y.float().cpu().numpy())).cuda().long()]
    assert torch.equal(lut[vp[at].long()], held(v.float() / sc[1][:, None]))
    x, tol = ref_head(k, w[1], cos[pos], sin[pos], norm, rope)
    s, got = sc[0].double()[:, None], lut[kp[at].long()]
    lo, hi = (held((x + sgn * tol) / s * (1 + sgn * 4 * U * torch.sign(x + sgn * tol))) for sgn in (-1, 1))
    assert ((x / s).abs() > 256).any()
    assert (got >= lo).all() and (got <= hi).all()
    ops.check_status()
