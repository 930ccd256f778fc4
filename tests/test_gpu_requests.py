"""GPU: cross-attention to encoder states of another length (sdmi_cross_attention) and adapters of many requests beside a shared
projection (sdmi_lora_gemm) against their definitions in 64 bits, element by element.

Tolerances, u = half a step of the 16-bit type (finfo.eps / 2), e = 2^-24 the same of fp32:
  attention  p is rounded to 16 bits (u p; below the type's smallest normal number half its smallest step, tiny * eps / 2), o once more
             (u |o|).  A score is off by at most (dim + 4) e sum |q||k| scale (fp32 sums of exact products, the scaling) and the base-2
             exponential by 4 e |score| (its argument's rounding) + 8 e, so every p is off by a factor of 1 +- r, r the sum of these; sums
             of up to nkv terms add (nkv + 64) e each, and an error of p goes into numerator and denominator.  With a = sum p |v| / sum p:
             tol = u (a + |o|) + (2 r + 2 (nkv + 64) e) (a + |o|) + nkv tiny eps / 2 max |v|.
  adapters   t is rounded to 16 bits (u |t|), out once (u |out|), the fp32 sums are off by (terms) e of the sums of absolute values:
             tol = u |out| + sum_r |b| (u |t| + tiny eps / 2 + 2 (k + 4) e scale sum |x||a|) + (k + rank + 8) e (sum |x||w| + sum |t||b| + |bias| + |residual|)."""
import math

import numpy as np
import pytest
import torch

from stable_diffusion_amd import engine as E, _lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
H16 = E.act_dtype() if torch.cuda.is_available() else torch.float16
U, TINY, E32 = torch.finfo(H16).eps / 2, torch.finfo(H16).tiny * torch.finfo(H16).eps / 2, 2.0 ** -24


def _h(rs, *shape, std=1.0):
    return torch.from_numpy((rs.standard_normal(shape) * std).astype(np.float32)).to(H16)


def _i32(v):
    return torch.tensor(v, dtype=torch.int64).to(torch.int32).to(DEV)


# ------------------------------------------------------------------------------------------------------------ attention
def _attention_oracle(q, k, v, heads, kvh, dim, scale, index, lens, qr, kr):
    """(o, tolerance) in 64 bits on the CPU, sample by sample and head by head; q (b, nq, heads * dim), k / v (contexts, nkv, kvh * dim)."""
    b, nq, nkv, n = q.shape[0], q.shape[1], k.shape[1], k.shape[0]
    o, tol = torch.zeros(b, nq, heads * dim, dtype=torch.float64), torch.zeros(b, nq, heads * dim, dtype=torch.float64)
    for i in range(b):
        c = index[i] if index is not None else (0 if n == 1 else i)
        if not 0 <= c < n:
            continue
        ln = min(max(lens[c], 0), nkv) if lens is not None else nkv
        seen = torch.ones(nq, ln, dtype=torch.bool)
        keys = torch.arange(ln)
        if qr is not None:
            seen = (qr[i][:, None] & kr[c][None, :ln]) != 0
            keys = torch.nonzero(kr[c][:ln] != 0).flatten()       # a key in no region may hold anything
            seen = seen[:, keys]
        if keys.numel() == 0:
            continue
        for h in range(heads):
            g = h * kvh // heads
            qd, kd, vd = q[i, :, h * dim:(h + 1) * dim].double(), k[c, keys, g * dim:(g + 1) * dim].double(), v[c, keys, g * dim:(g + 1) * dim].double()
            s = scale * (qd @ kd.t())
            r = (dim + 4) * E32 * scale * (qd.abs() @ kd.abs().t()) + 4 * E32 * (s.abs() + s.abs().amax(1, keepdim=True)) + 8 * E32
            r = r.masked_fill(~seen, 0.0).amax(1, keepdim=True) if keys.numel() else 0.0
            p = torch.exp(s - s.masked_fill(~seen, -math.inf).amax(1, keepdim=True).clamp_min(-1e30)).masked_fill(~seen, 0.0)
            l = p.sum(1, keepdim=True)
            l = torch.where(l == 0, torch.ones_like(l), l)
            oo, aa = p @ vd / l, p @ vd.abs() / l
            o[i, :, h * dim:(h + 1) * dim] = oo
            t = U * (aa + oo.abs()) + (2 * r + 2 * (ln + 64) * E32) * (aa + oo.abs()) + ln * TINY * float(vd.abs().max())
            tol[i, :, h * dim:(h + 1) * dim] = torch.where(seen.any(1, keepdim=True), t, torch.zeros_like(t))
    return o, tol


def _close(got, want, tol, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    bad = (got - want).abs() > tol
    print("%s: max error / tolerance %.3f" % (what, float(((got - want).abs() / tol.clamp_min(1e-300)).max())), flush=True)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()), torch.nonzero(bad)[:4].tolist())


def _attention_case(seed, batch, contexts, heads, kvh, dim, nq, nkv, index=None, lens=None, regions=0, nan=True, std=1.5):
    rs = np.random.RandomState(seed)
    q, k, v = _h(rs, batch, nq, heads * dim, std=std), _h(rs, contexts, nkv, kvh * dim), _h(rs, contexts, nkv, kvh * dim)
    qr = kr = None
    if regions:
        bits = lambda *s: torch.from_numpy(((1 << rs.randint(0, regions, s).astype(np.int64)) * rs.randint(0, 4, s).clip(0, 1)).astype(np.uint32).view(np.int32))
        qr, kr = bits(batch, nq), bits(contexts, nkv)
    # what lies past a context's end, or in no region, is anything
    kd, vd = k.clone(), v.clone()
    if nan:
        for c in range(contexts):
            dead = torch.zeros(nkv, dtype=torch.bool)
            if lens is not None:
                dead[min(max(lens[c], 0), nkv):] = True
            if kr is not None:
                dead |= kr[c] == 0
            kd[c][dead], vd[c][dead] = float("nan"), float("inf")
    return q, k, v, kd, vd, qr, kr


def _run_attention(q, kd, vd, heads, kvh, dim, index, lens, qr, kr, scale=None, out=None):
    """k and v as neighbouring column ranges of one wider buffer, q as the middle of another."""
    b, nq, n, nkv = q.shape[0], q.shape[1], kd.shape[0], kd.shape[1]
    w = kvh * dim
    kv = torch.full((n, nkv, 2 * w + 16), float("nan"), dtype=H16)
    kv[..., 8:8 + w], kv[..., 8 + w:8 + 2 * w] = kd, vd
    qb = torch.full((b, nq, heads * dim + 24), float("nan"), dtype=H16)
    qb[..., 16:16 + heads * dim] = q
    kva, qa = E.Act(kv.to(DEV), n, 1, nkv, 2 * w + 16), E.Act(qb.to(DEV), b, 1, nq, heads * dim + 24)
    o = E.cross_attention(qa.cols(16, heads * dim), kva.cols(8, w), kva.cols(8 + w, w), heads, kv_heads=kvh, dim=dim, scale=scale,
                          index=None if index is None else _i32(index), lens=None if lens is None else _i32(lens),
                          query_regions=None if qr is None else qr.to(DEV), key_regions=None if kr is None else kr.to(DEV), out=out)
    return o.buf if out is None else o


ATT = [  # batch, contexts, heads, kv heads, dim, nq, nkv, index, lens, regions
    (1, 1, 1, 1, 64, 1, 1, None, None, 0),
    (2, 2, 2, 2, 64, 130, 77, None, [77, 1], 0),
    (3, 1, 2, 2, 64, 65, 64, None, [63], 0),
    (3, 2, 2, 1, 64, 129, 65, [1, 0, 1], [65, 0], 0),
    (2, 2, 5, 5, 64, 200, 231, None, [200, 129], 0),
    (4, 3, 4, 2, 40, 33, 100, [2, 2, 0, 1], [100, 64, 65], 0),
    (2, 2, 3, 3, 8, 70, 9, None, None, 0),
    (1, 1, 2, 2, 32, 300, 128, None, None, 0),
    (2, 2, 2, 2, 72, 97, 127, None, [127, 128], 0),
    (2, 2, 8, 8, 80, 101, 133, None, [133, -5], 0),
    (2, 2, 2, 2, 96, 131, 190, None, [1000, 3], 0),
    (2, 2, 4, 1, 128, 66, 257, None, None, 0),
    (2, 2, 2, 2, 160, 140, 130, None, [130, 66], 0),
    (2, 2, 2, 2, 200, 140, 70, None, None, 0),
    (2, 2, 2, 1, 256, 150, 193, None, [150, 193], 0),
    # few rows: one wave tile for four waves; long keys in pieces
    (2, 2, 4, 4, 64, 1, 5, None, [5, 0], 0),
    (3, 3, 8, 2, 64, 1, 1025, None, [1025, 1, 128], 0),
    (2, 2, 16, 2, 128, 1, 2000, None, [1999, 130], 0),
    (2, 2, 2, 2, 256, 7, 700, None, [700, 0], 0),
    (1, 1, 2, 2, 160, 40, 1111, None, None, 0),
    (2, 3, 2, 2, 32, 64, 4099, [2, 0], [4099, 7, 4001], 0),
    (1, 1, 2, 2, 64, 144, 3001, None, None, 0),
    (1, 1, 1, 1, 96, 129, 1500, None, [1409], 0),
    # regions
    (2, 2, 2, 2, 64, 150, 154, None, None, 3),
    (2, 1, 4, 2, 64, 9, 600, None, [599], 32),
    (2, 2, 2, 2, 80, 131, 90, [1, 1], [0, 90], 32),
    (1, 1, 2, 2, 256, 3, 900, None, None, 2),
    (2, 2, 2, 1, 160, 70, 65, None, None, 4),
    (2, 2, 2, 2, 96, 140, 2100, None, [2100, 1], 2),
    (1, 1, 2, 2, 128, 140, 300, None, None, 32),
    (1, 1, 2, 2, 32, 140, 300, None, None, 32),
]


@pytest.mark.parametrize("case", range(len(ATT)))
def test_attention(case):
    batch, contexts, heads, kvh, dim, nq, nkv, index, lens, regions = ATT[case]
    q, k, v, kd, vd, qr, kr = _attention_case(case, batch, contexts, heads, kvh, dim, nq, nkv, index, lens, regions)
    got = _run_attention(q, kd, vd, heads, kvh, dim, index, lens, qr, kr)
    want, tol = _attention_oracle(q, k, v, heads, kvh, dim, dim ** -0.5, index, lens, qr, kr)
    _close(got, want, tol, "attention %s" % (ATT[case],))


@pytest.mark.parametrize("nq,nkv", [(200, 100), (1, 2000)])
def test_attention_large_scores_and_other_scale(nq, nkv):
    """Scores of some hundreds (one key takes it all) and a scale of the caller's."""
    q, k, v, kd, vd, _, _ = _attention_case(77, 2, 2, 2, 2, 64, nq, nkv, std=60.0)
    got = _run_attention(q, kd, vd, 2, 2, 64, None, None, None, None, scale=0.3)
    want, tol = _attention_oracle(q, k, v, 2, 2, 64, float(np.float32(0.3)), None, None, None, None)
    _close(got, want, tol, "attention, scores of hundreds")


@pytest.mark.parametrize("nq,nkv", [(1, 6000), (200, 6000), (200, 900)])
@pytest.mark.parametrize("far", [12.0, 16.0, 20.0])
def test_attention_small_weights_add_up(nq, nkv, far):
    """One key far above thousands whose p = 2^-far is at or below the 16-bit type's smallest normal number: they count, in the
    numerator and in the sum."""
    rs = np.random.RandomState(int(far))
    q, k, v = torch.zeros(1, nq, 64), torch.zeros(1, nkv, 64), _h(rs, 1, nkv, 64)
    q[:, :, 0], k[:, nkv // 2, 0] = 1.0, 1.0
    v[:, :, 0] = 1.0                                         # column 0 comes out as 1 if and only if both agree
    q, k = q.to(H16), k.to(H16)
    got = _run_attention(q, k, v, 1, 1, 64, None, None, None, None, scale=far * math.log(2.0))
    want, tol = _attention_oracle(q, k, v, 1, 1, 64, float(np.float32(far * math.log(2.0))), None, None, None, None)
    _close(got, want, tol, "attention, %d weights of 2^-%g" % (nkv, far))


@pytest.mark.parametrize("nq", [3, 200])
def test_attention_no_keys_gives_zeros(nq):
    q = _h(np.random.RandomState(1), 2, nq, 128)
    qa, kv = E.Act(q.to(DEV), 2, 1, nq, 128), E.Act(torch.empty((2, 0, 128), dtype=H16, device=DEV), 2, 1, 0, 128)
    assert not E.cross_attention(qa, kv, kv, 2).buf.any()
    kv = E.Act(torch.full((2, 90, 128), float("nan"), dtype=H16, device=DEV), 2, 1, 90, 128)
    assert not E.cross_attention(qa, kv, kv, 2, index=_i32([-1, 2])).buf.any()          # no such context
    assert not E.cross_attention(qa, kv, kv, 2, lens=_i32([0, -3])).buf.any()
    sets = dict(query_regions=_i32([[1] * nq] * 2), key_regions=_i32([[0] * 90] * 2))
    assert not E.cross_attention(qa, kv, kv, 2, **sets).buf.any()


@pytest.mark.parametrize("nq,nkv", [(37, 77), (130, 77), (5, 1500)])
def test_attention_writes_its_own_columns_only(nq, nkv):
    q, k, v, kd, vd, _, _ = _attention_case(5, 2, 2, 2, 2, 40, nq, nkv, lens=[nkv, 3])
    buf = torch.full((2, nq, 96), 7.0, dtype=H16, device=DEV)
    out = E.Act(buf, 2, 1, nq, 96).cols(8, 80)
    _run_attention(q, kd, vd, 2, 2, 40, None, [nkv, 3], None, None, out=out)
    want, tol = _attention_oracle(q, k, v, 2, 2, 40, 40 ** -0.5, None, [nkv, 3], None, None)
    _close(buf[..., 8:88], want, tol, "attention into a view")
    assert bool((buf[..., :8] == 7.0).all()) and bool((buf[..., 88:] == 7.0).all())


@pytest.mark.parametrize("dim,off", [(64, 4), (40, 12), (256, 4), (32, 20), (96, 0), (160, 4)])
def test_attention_rows_start_anywhere_on_8_bytes(dim, off):
    q, k, v, kd, vd, _, _ = _attention_case(31, 2, 2, 2, 1, dim, 100, 77, lens=[77, 0])
    buf = torch.full((2, 100, 2 * dim + 28), 3.0, dtype=H16, device=DEV)
    _run_attention(q, kd, vd, 2, 1, dim, None, [77, 0], None, None, out=E.Act(buf, 2, 1, 100, 2 * dim + 28).cols(off, 2 * dim))
    want, tol = _attention_oracle(q, k, v, 2, 1, dim, dim ** -0.5, None, [77, 0], None, None)
    _close(buf[..., off:off + 2 * dim], want, tol, "attention, %d wide from column %d" % (dim, off))
    assert bool((buf[..., :off] == 3.0).all()) and bool((buf[..., off + 2 * dim:] == 3.0).all())


def test_attention_offsets_past_32_bits():
    """Rows 128 KB apart (the last one 5 GB behind the first) and contexts further still."""
    nkv, ld = 40000, 1 << 16
    rs = np.random.RandomState(3)
    base = torch.empty((nkv, ld), dtype=H16, device=DEV)
    k, v, q = _h(rs, 1, nkv, 64), _h(rs, 1, nkv, 64), _h(rs, 2, 1, 64)
    base[:, :64], base[:, 64:128] = k[0].to(DEV), v[0].to(DEV)
    qd, o = q.to(DEV), torch.empty((2, 1, 64), dtype=H16, device=DEV)
    ws = torch.empty((L.load().sdmi_cross_attention_ws_bytes(2, 1, 1, 64, 1, nkv),), dtype=torch.uint8, device=DEV)
    # two contexts: rows 0.. and rows 20000.. of the same memory
    L.call("sdmi_cross_attention", qd.data_ptr(), 64, 64, base.data_ptr(), ld, 20000 * ld, base.data_ptr() + 128, ld, 20000 * ld, o.data_ptr(), 64, 64, 2, 2, 1, 1, 64, 1,
           20000, 0, 0, 0, 0, 0, 0, 0.125, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    want, tol = _attention_oracle(q, k.view(2, 20000, 64), v.view(2, 20000, 64), 1, 1, 64, 0.125, None, None, None, None)
    _close(o, want, tol, "attention over 5 GB of rows")


def test_attention_without_workspace_is_not_cut():
    q, k, v, kd, vd, _, _ = _attention_case(8, 2, 2, 2, 2, 64, 1, 3000)
    qa, ka, va, o = (t.to(DEV) for t in (q, kd, vd, torch.empty_like(q)))
    assert L.load().sdmi_cross_attention_ws_bytes(2, 2, 2, 64, 1, 3000) > 0
    L.call("sdmi_cross_attention", qa.data_ptr(), 128, 128, ka.data_ptr(), 128, 128 * 3000, va.data_ptr(), 128, 128 * 3000, o.data_ptr(), 128, 128, 2, 2, 2, 2, 64, 1, 3000,
           0, 0, 0, 0, 0, 0, 0.125, 0, 0, torch.cuda.current_stream().cuda_stream)
    want, tol = _attention_oracle(q, k, v, 2, 2, 64, 0.125, None, None, None, None)
    _close(o, want, tol, "attention without a workspace")


ATT_WIDTHS = [  # the two block shapes at every width, with regions as well
    (2, 2, 2, 2, 32, 5, 700, [1, 1], [3, 650], 3),
    (2, 2, 2, 1, 128, 20, 130, None, [129, 130], 3),
    (2, 1, 2, 2, 160, 30, 700, None, [641], 3),
    (1, 1, 3, 3, 256, 90, 140, None, None, 3),
    (2, 2, 2, 2, 96, 20, 70, None, [70, 33], 0),
    (1, 1, 2, 2, 32, 200, 1100, None, None, 0),
    (2, 2, 2, 2, 104, 200, 600, [1, 1], [5, 577], 0),
    (1, 1, 1, 1, 248, 65, 1000, None, None, 0),
]


@pytest.mark.parametrize("case", range(len(ATT_WIDTHS)))
def test_attention_block_shapes(case):
    batch, contexts, heads, kvh, dim, nq, nkv, index, lens, regions = ATT_WIDTHS[case]
    q, k, v, kd, vd, qr, kr = _attention_case(200 + case, batch, contexts, heads, kvh, dim, nq, nkv, index, lens, regions)
    got = _run_attention(q, kd, vd, heads, kvh, dim, index, lens, qr, kr)
    want, tol = _attention_oracle(q, k, v, heads, kvh, dim, dim ** -0.5, index, lens, qr, kr)
    _close(got, want, tol, "attention %s" % (ATT_WIDTHS[case],))


def test_attention_refuses_tensors_of_another_kind():
    a = E.Act(torch.zeros((2, 8, 64), dtype=H16, device=DEV), 2, 1, 8, 64)
    sets = torch.zeros((2, 8), dtype=torch.int32, device=DEV)
    for kw in (dict(lens=torch.zeros(2, dtype=torch.int32)), dict(lens=_i32([1, 2]).long()), dict(lens=_i32([1])), dict(index=_i32([[0, 1]])),
               dict(query_regions=sets), dict(query_regions=sets, key_regions=sets[:, ::2]), dict(index=_i32([0, 9, 1, 9])[::2])):
        with pytest.raises(L.SdmiError):
            E.cross_attention(a, a, a, 1, **kw)
    host = E.Act(torch.zeros((2, 8, 64), dtype=H16), 2, 1, 8, 64)
    for q, k in ((a, host), (host, a), (host, host)):
        with pytest.raises(L.SdmiError):
            E.cross_attention(q, k, k, 1)
    with pytest.raises(L.SdmiError):
        E.cross_attention(a, a.cols(0, 32), a, 1)
    both = E.Act(torch.zeros((2, 8, 192), dtype=H16, device=DEV), 2, 1, 8, 192)
    for out in (a, both.cols(32, 64), both.cols(127, 64)):
        with pytest.raises(L.SdmiError, match="memory"):
            E.cross_attention(a if out is a else both.cols(0, 64), both.cols(64, 64), both.cols(128, 64), 1, out=out)
    wide = E.Act(a.buf.float(), 2, 1, 8, 64)
    for q, k, out in ((wide, a, None), (a, wide, None), (a, a, wide)):
        with pytest.raises(L.SdmiError):
            E.cross_attention(q, k, k, 1, out=out)


FAR = [  # nq, nkv, dim, regions: a wave with a share of the tile or all of it, one partial tile, keys in pieces
    (1, 1, 64, 0), (200, 1, 64, 0), (200, 77, 64, 0), (5, 77, 64, 0), (130, 600, 64, 0), (1, 2000, 64, 0), (70, 130, 32, 0), (100, 200, 96, 0), (3, 900, 128, 0),
    (90, 140, 160, 0), (66, 100, 256, 0), (200, 154, 64, 3), (9, 600, 64, 3)]


@pytest.mark.parametrize("x,y,scale", [(60000.0, 60000.0, None), (30000.0, 50000.0, None), (3.0, 2.0, 1e9), (100.0, -90.0, 1e9), (1.5, 1.25, 1e15), (0.75, -0.5, 1e15)])
@pytest.mark.parametrize("nq,nkv,dim,regions", FAR)
def test_attention_scores_far_apart(nq, nkv, dim, regions, x, y, scale):
    """Scores up to 2^60 in magnitude, each row's best one ahead of the next by 2^64 or more in weight: its value comes out, to the bit.
    Every score is one product, exact in fp32."""
    rs = np.random.RandomState(nq + nkv + dim)
    q, k, v = torch.zeros(1, nq, dim), torch.zeros(1, nkv, dim), _h(rs, 1, nkv, dim)
    q[0, torch.arange(nq), torch.arange(nq) % dim] = x
    # of the keys that meet a query, one after the other a step of the 16-bit type nearer to y
    rank = torch.from_numpy(np.argsort(rs.rand(dim, nkv), 1)).t()
    k[0] = (y * (1 - torch.clamp(rank, max=12) * 2 * U)).to(H16).float()
    k[0][rank > 12] = float(-y)
    q, k = q.to(H16), k.to(H16)
    qr = kr = None
    seen = torch.ones(nq, nkv, dtype=torch.bool)
    if regions:
        qr, kr = torch.from_numpy(rs.randint(0, 8, (1, nq))).to(torch.int32), torch.from_numpy(rs.randint(1, 8, (1, nkv))).to(torch.int32)
        seen = (qr[0][:, None] & kr[0][None]) != 0
    s = (q[0].double() @ k[0].double().t()).masked_fill(~seen, -math.inf)
    top = s.topk(min(2, nkv), 1).values
    ahead = top[:, 0] - top[:, -1] if nkv > 1 else torch.full((nq,), math.inf, dtype=torch.float64)
    got = _run_attention(q, k, v, 1, 1, dim, None, None, qr, kr, scale=scale)[0].cpu()
    for i in range(nq):
        if not seen[i].any():
            assert not got[i].any(), i
        elif float(ahead[i]) * (dim ** -0.5 if scale is None else scale) > 64:
            assert torch.equal(got[i], v[0, int(s[i].argmax())]), (i, got[i][:4], v[0, int(s[i].argmax())][:4])
        else:                                               # a tie: neither of the values may be lost
            best = torch.nonzero(s[i] == top[i, 0]).flatten()
            mean = v[0, best].double().mean(0)
            assert bool(((got[i].double() - mean).abs() <= 2 * U * mean.abs() + U * v[0, best].double().abs().mean(0) + TINY).all()), i


@pytest.mark.parametrize("e", [-8, -5, -4, -3, 0, 4, 8, 12, 24])
@pytest.mark.parametrize("nq,nkv,dim", [(200, 90, 64), (4, 90, 64), (3, 1500, 64), (130, 700, 64), (100, 150, 128), (2, 1000, 256)])
def test_attention_near_ties_of_large_scores(nq, nkv, dim, e):
    """Scores of 2^20 + d, d = 0, 1/8, ... 8, times 2^e: exact in fp32, so the weights are 2^-((8 - d) 2^e) however large they are.
    The scale's rounding and log2(e)'s move an exponent by 2^-22 of itself at most (20 times that where the weight still counts)."""
    rs = np.random.RandomState(e + 50)
    q, k, v = torch.zeros(1, nq, dim), torch.zeros(1, nkv, dim), _h(rs, 1, nkv, dim)
    d = torch.from_numpy(rs.randint(0, 65, nkv)) / 8.0
    q[..., 0], q[..., 1], k[..., 0], k[0, :, 1] = 1024.0, 1.0, 1024.0, d.float()
    scale = float(np.float32(math.log(2.0) * 2.0 ** e))
    got = _run_attention(q.to(H16), k.to(H16), v, 1, 1, dim, None, None, None, None, scale=scale)
    p = torch.exp2((d - d.max()).double() * (scale / math.log(2.0)))
    o, a = p @ v[0].double() / p.sum(), p @ v[0].double().abs() / p.sum()
    r = 20 * 2.0 ** -22 + 16 * E32
    tol = U * (a + o.abs()) + (2 * r + 2 * (nkv + 64) * E32) * (a + o.abs()) + nkv * TINY * float(v.double().abs().max())
    _close(got, o.expand(1, nq, dim), tol.expand(1, nq, dim), "attention, near ties of 2^%d" % (20 + e))


@pytest.mark.skipif(H16 is torch.float16, reason="dot products of fp16 cannot lie past 2^40")
@pytest.mark.parametrize("nq,nkv", [(200, 77), (2, 50), (1, 1500), (130, 700)])
@pytest.mark.parametrize("x,y", [(2.0 ** 60, -2.0 ** 60), (-2.0 ** 50, 2.0 ** 60), (2.0 ** 60, 2.0 ** 60), (2.0 ** 62, -2.0 ** 64)])
def test_attention_of_bf16_rows_far_from_zero(nq, nkv, x, y):
    """Every score of a row past 1e30 in magnitude (down to -1e38): the mean of the values."""
    q, k, v = torch.zeros(1, nq, 64), torch.zeros(1, nkv, 64), _h(np.random.RandomState(1), 1, nkv, 64)
    q[..., 0], k[..., 0] = x, y
    got = _run_attention(q.to(H16), k.to(H16), v, 1, 1, 64, None, None, None, None)
    mean, mag = v[0].double().mean(0), v[0].double().abs().mean(0)
    tol = U * mean.abs() + 2 * (nkv + 64) * E32 * mag
    _close(got, mean.expand(1, nq, 64), tol.expand(1, nq, 64), "attention, rows of scores %g" % (x * y))


# ------------------------------------------------------------------------------------------------------------ adapters
def _lora_oracle(x, w, a, b, scale, ids, per, groups, bias, residual):
    x, w, a, b = x.double(), w.double(), a.double(), b.double()
    m, n, r = x.shape[0], w.shape[0], b.shape[2]
    out, mag = x @ w.t(), x.abs() @ w.abs().t()
    extra = torch.zeros_like(out)
    for i in range(m):
        j = ids[i // per]
        if not 0 <= j < a.shape[0]:
            continue
        sc = float(scale[j])
        t, ta = sc * (a[j] @ x[i]), sc * (a[j].abs() @ x[i].abs())
        for g in range(groups):
            c = slice(g * n // groups, (g + 1) * n // groups)
            tg, tag = t[g * r:(g + 1) * r], ta[g * r:(g + 1) * r]
            out[i, c] += b[j, c] @ tg
            mag[i, c] += b[j, c].abs() @ tg.abs()
            extra[i, c] = b[j, c].abs() @ (U * tg.abs() + TINY + 2 * (x.shape[1] + 4) * E32 * tag)
    if bias is not None:
        out, mag = out + bias.double(), mag + bias.double().abs()
    if residual is not None:
        out, mag = out + residual.double(), mag + residual.double().abs()
    return out, U * out.abs() + TINY + extra + (x.shape[1] + r + 8) * E32 * mag


def _lora_case(seed, m, k, n, groups, rank, adapters, bias, residual):
    rs = np.random.RandomState(seed)
    x, w, a, b = _h(rs, m, k), _h(rs, n, k, std=k ** -0.5), _h(rs, adapters, groups * rank, k, std=k ** -0.5), _h(rs, adapters, n, rank, std=rank ** -0.5)
    scale = torch.from_numpy((rs.rand(adapters) * 2 - 0.5).astype(np.float32))
    return x, w, a, b, scale, torch.from_numpy(rs.randn(n).astype(np.float32)) if bias else None, _h(rs, m, n) if residual else None


def _run_lora(x, w, a, b, scale, ids, bias, residual, out=None):
    m, k, n = x.shape[0], x.shape[1], w.shape[0]
    xb = torch.full((1, m, k + 16), float("nan"), dtype=H16)
    xb[0, :, 8:8 + k] = x
    res = None if residual is None else E.Act(residual.to(DEV).view(1, m, n), 1, 1, m, n)
    y = E.lora_gemm(E.Act(xb.to(DEV), 1, 1, m, k + 16).cols(8, k), w.to(DEV), n, E.LoraPack(a.to(DEV), b.to(DEV), scale.to(DEV)), _i32(ids),
                    bias=None if bias is None else bias.to(DEV), residual=res, out=out)
    return y.buf.view(m, -1) if out is None else y


LORA = [  # rows per id, ids, k, n, groups, rank, adapters, bias, residual
    (1, [0], 8, 8, 1, 8, 1, False, False),
    (1, [2], 1024, 1024, 1, 16, 4, True, True),
    (1, [1, 0, -1, 3, 1], 72, 40, 1, 8, 3, True, False),
    (7, [1, 0, 2], 320, 320, 1, 16, 3, True, True),
    (64, [0, 1], 64, 128, 1, 32, 2, False, False),
    (100, [1, 1, 0], 136, 104, 1, 24, 2, True, False),
    (130, [0], 640, 120, 3, 8, 1, False, False),
    (77, [3, -1, 0, 1], 192, 984, 3, 16, 4, True, True),
    (33, [1, 0], 200, 72, 3, 40, 2, False, True),
    (1, list(range(64)), 128, 256, 1, 32, 64, True, False),
    (1, [(i * 7) % 5 - 1 for i in range(205)], 256, 192, 1, 128, 4, True, True),
    (1, [(i * i) % 97 for i in range(150)], 88, 72, 1, 8, 97, False, False),
    (3, [(i * 5) % 9 for i in range(50)], 104, 176, 2, 16, 9, False, True),
    (300, [-1, 5], 96, 64, 1, 16, 5, True, False),
    (1, [2 ** 31 - 1, -2 ** 31, 0, 1], 64, 64, 1, 256, 1, False, False),
    (900, [1, 0], 64, 64, 1, 64, 2, True, True),
    (2304, [0, 1], 64, 1920, 3, 8, 2, False, False),
    (1, [0] * 17, 5120, 16, 1, 8, 1, True, False),
]


@pytest.mark.parametrize("case", range(len(LORA)))
def test_lora(case):
    per, ids, k, n, groups, rank, adapters, bias, residual = LORA[case]
    x, w, a, b, scale, bi, res = _lora_case(case, per * len(ids), k, n, groups, rank, adapters, bias, residual)
    got = _run_lora(x, w, a, b, scale, ids, bi, res)
    want, tol = _lora_oracle(x, w, a, b, scale, ids, per, groups, bi, res)
    _close(got, want, tol, "lora %s" % ((per, len(ids)) + LORA[case][2:],))


LORA_KINDS = [  # what the larger kernels and the ranks beyond their first tile do
    (1, [i % 3 for i in range(12)], 136, 56, 1, 16, 3, True, True),
    (4096, [1, 0], 72, 2048, 1, 16, 2, True, False),
    (4096, [0, -1], 64, 2064, 2, 32, 1, False, True),
    (2048, [1, 0], 72, 1032, 1, 8, 2, True, True),
    (1000, [1, 0, 1, -1], 64, 1080, 3, 24, 2, True, False),
    (2050, [0, 1], 64, 1024, 1, 40, 2, False, True),
    (4100, [0, 1], 72, 512, 2, 64, 2, True, False),
    (16, [(i * 7) % 9 - 1 for i in range(256)], 64, 1032, 1, 16, 8, False, True),
    (1, [(i * i) % 11 for i in range(4100)], 64, 1080, 3, 72, 10, True, False),
    (65, [1, 0, -1, 1], 328, 40, 1, 256, 2, False, False),
    (33, [(i * 5) % 7 - 1 for i in range(130)], 72, 136, 1, 16, 6, False, True),        # rows taken in the order of their adapters, past one chunk of them
    (1, [(i * 389) % 1100 for i in range(300)], 64, 72, 1, 8, 1100, True, False),       # too many adapters to order
    (1, [(i * 389) % 1023 for i in range(300)], 64, 72, 1, 8, 1023, True, False),
    (1, [-1, 7] * 40, 64, 72, 1, 8, 7, True, True),
    (1, [2] * 65 + [0] * 63 + [1] + [2] * 64, 64, 80, 2, 24, 3, False, False),
]


@pytest.mark.parametrize("case", range(len(LORA_KINDS)))
def test_lora_kinds(case):
    per, ids, k, n, groups, rank, adapters, bias, residual = LORA_KINDS[case]
    x, w, a, b, scale, bi, res = _lora_case(100 + case, per * len(ids), k, n, groups, rank, adapters, bias, residual)
    got = _run_lora(x, w, a, b, scale, ids, bi, res)
    want, tol = _lora_oracle(x, w, a, b, scale, ids, per, groups, bi, res)
    _close(got, want, tol, "lora %s" % ((per, len(ids)) + LORA_KINDS[case][2:],))


def _lora_oracle_by_id(x, w, a, b, scale, ids, per, groups, bias, residual):
    """_lora_oracle, all rows of an adapter at once."""
    x, w, a, b = x.double(), w.double(), a.double(), b.double()
    m, n, r, k = x.shape[0], w.shape[0], b.shape[2], x.shape[1]
    out, mag, extra = x @ w.t(), x.abs() @ w.abs().t(), torch.zeros(m, n, dtype=torch.float64)
    row_id = torch.tensor(ids).repeat_interleave(per)
    for j in sorted({i for i in ids if 0 <= i < a.shape[0]}):
        rows, sc = torch.nonzero(row_id == j).flatten(), float(scale[j])
        t, ta = sc * (x[rows] @ a[j].t()), abs(sc) * (x[rows].abs() @ a[j].abs().t())
        for g in range(groups):
            c, gr = slice(g * n // groups, (g + 1) * n // groups), slice(g * r, (g + 1) * r)
            out[rows, c] += t[:, gr] @ b[j, c].t()
            mag[rows, c] += t[:, gr].abs() @ b[j, c].abs().t()
            extra[rows, c] = (U * t[:, gr].abs() + TINY + 2 * (k + 4) * E32 * ta[:, gr]) @ b[j, c].abs().t()
    if bias is not None:
        out, mag = out + bias.double(), mag + bias.double().abs()
    if residual is not None:
        out, mag = out + residual.double(), mag + residual.double().abs()
    return out, U * out.abs() + TINY + extra + (k + r + 8) * E32 * mag


LORA_LONG = [  # every ring and panel refilled several times, the last step of K a partial one
    # rows per id, ids, k, n, groups, rank, adapters, bias, residual, kernel
    (4096, [1, 0], 392, 2048, 1, 16, 2, True, False, "lora_gemm_kernel<128, 128, false, 16>"),
    (4096, [1, -1], 392, 2048, 1, 32, 2, False, True, "lora_gemm_kernel<128, 128, false, 32>"),
    (2048, [1, 0], 456, 1032, 1, 8, 2, False, True, "lora_gemm_kernel<128, 64, false, 16>"),
    (2048, [0, 1], 456, 1032, 1, 24, 2, True, False, "lora_gemm_kernel<128, 64, false, 32>"),
    (600, [0, 1], 648, 136, 1, 16, 2, True, True, "lora_gemm_kernel<64, 64, false, 16>"),
    (600, [1, 0], 520, 1080, 3, 32, 2, False, False, "lora_gemm_kernel<64, 64, false, 32>"),
    (576, [0, 1], 648, 136, 1, 64, 2, True, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, false, 0>"),
    (600, [1, -1, 0], 520, 264, 3, 72, 2, False, True, "lora_shrink_kernel + lora_gemm_kernel<64, 64, false, 0>"),
    (2048, [1, 0], 456, 1032, 1, 200, 2, False, False, "lora_shrink_kernel + lora_gemm_kernel<128, 64, false, 0>"),
    (1, [(i * i) % 6 - 1 for i in range(1155)], 648, 200, 1, 72, 5, True, True, "lora_shrink_kernel + lora_gemm_kernel<64, 64, true, 0>"),
    (16, [(i * 7) % 9 - 1 for i in range(256)], 520, 1040, 2, 40, 8, False, False, "lora_shrink_kernel + lora_gemm_kernel<128, 64, true, 0>"),
    (1, [(i * 3) % 5 - 1 for i in range(40)], 2056, 72, 1, 32, 4, True, False, "lora_shrink_kernel + lora_rows_kernel<4, false>"),
    (2, [(i * 3) % 5 - 1 for i in range(15)], 3080, 72, 1, 40, 4, False, True, "lora_shrink_kernel + lora_rows_kernel<2, false>"),
    (1, [(i * 3) % 5 - 1 for i in range(12)], 4104, 40, 1, 16, 4, True, True, "lora_shrink_kernel + lora_rows_kernel<1, false>"),
    (1, [1, 0, -1], 5000, 72, 1, 16, 2, True, False, "lora_rows_kernel<1, true>"),
    # the low-rank factor by blocks of 64, 32 and 16 rows
    (4096, [1, 0], 1160, 64, 1, 64, 2, False, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, false, 0>"),
    (1152, [0, 1], 2056, 72, 1, 64, 2, True, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, false, 0>"),
    (1, [(i * i) % 6 - 1 for i in range(2100)], 1096, 72, 1, 56, 5, False, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, true, 0>"),
    (1, [(i * 7) % 3 for i in range(500)], 2120, 72, 1, 24, 3, False, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, true, 0>"),
    (1, [(i * 7) % 3 for i in range(70)], 4104, 72, 1, 8, 3, False, False, "lora_shrink_kernel + lora_gemm_kernel<64, 64, true, 0>"),
]


@pytest.mark.parametrize("case", range(len(LORA_LONG)))
def test_lora_many_steps(case):
    per, ids, k, n, groups, rank, adapters, bias, residual, kernel = LORA_LONG[case]
    x, w, a, b, scale, bi, res = _lora_case(300 + case, per * len(ids), k, n, groups, rank, adapters, bias, residual)
    got = _run_lora(x, w, a, b, scale, ids, bi, res)
    ran = L.load().sdmi_last_kernel().decode()
    assert ran == kernel
    want, tol = _lora_oracle_by_id(x, w, a, b, scale, ids, per, groups, bi, res)
    _close(got, want, tol, "lora %s" % ((per, len(ids)) + LORA_LONG[case][2:],))


def test_the_two_forms_of_the_oracle_agree():
    args = _lora_case(5, 60, 40, 48, 3, 8, 3, True, True)
    a, b = (f(*args[:5], [0, -1, 2, 3, 1, 2], 10, 3, *args[5:]) for f in (_lora_oracle, _lora_oracle_by_id))
    assert torch.allclose(a[0], b[0], rtol=1e-12, atol=1e-12)
    assert (b[1] >= a[1] - 1e-12).all()                     # a negative scale's bound is its size


@pytest.mark.parametrize("m", [3, 40, 200, 1000])
def test_lora_one_id_for_any_number_of_rows(m):
    x, w, a, b, scale, _, _ = _lora_case(9, m, 64, 72, 1, 16, 3, False, False)
    xd, wd, ad, bd, sd, idd = x.to(DEV), w.to(DEV), a.to(DEV), b.to(DEV), scale.to(DEV), _i32([2])
    out = torch.empty((m, 72), dtype=H16, device=DEV)
    ws = torch.empty((max(L.load().sdmi_lora_gemm_ws_bytes(m, 72, 64, 16, 1, 2 ** 31 - 1), 2) // 2,), dtype=H16, device=DEV)
    L.call("sdmi_lora_gemm", xd.data_ptr(), 64, wd.data_ptr(), 64, out.data_ptr(), 72, m, 72, 64, 0, 0, 0, ad.data_ptr(), bd.data_ptr(), sd.data_ptr(), 3, 16, 1,
           idd.data_ptr(), 2 ** 31 - 1, 0, ws.data_ptr(), 2 * ws.numel(), torch.cuda.current_stream().cuda_stream)
    want, tol = _lora_oracle(x, w, a, b, scale, [2], m, 1, None, None)
    _close(out, want, tol, "lora, %d rows of one request" % m)


def test_lora_refuses_tensors_of_another_kind():
    x, w, a, b, scale, _, _ = _lora_case(9, 24, 64, 72, 1, 16, 3, False, False)
    xa, wd, pack = E.Act(x.to(DEV).view(1, 24, 64), 1, 1, 24, 64), w.to(DEV), E.LoraPack(a.to(DEV), b.to(DEV), scale.to(DEV))
    good = dict(lora=pack, ids=_i32([0, 1]))
    E.lora_gemm(xa, wd, 72, **good)
    for kw in (dict(ids=_i32([0] * 5)), dict(ids=_i32([0, 1]).long()), dict(ids=torch.zeros(2, dtype=torch.int32)), dict(ids=_i32([])),
               dict(lora=E.LoraPack(a, b, scale)), dict(bias=torch.zeros(72, dtype=H16, device=DEV)), dict(bias=torch.zeros(64, device=DEV)),
               dict(residual=xa), dict(out=xa)):
        with pytest.raises(L.SdmiError):
            E.lora_gemm(xa, wd, 72, **{**good, **kw})
    square = torch.zeros((64, 64), dtype=H16, device=DEV)
    with pytest.raises(L.SdmiError, match="memory"):
        E.lora_gemm(xa, square, 64, E.LoraPack(pack.a, pack.b[:, :64].contiguous(), pack.scale), good["ids"], out=xa)
    for x2, w2, n in ((xa, wd.t(), 64), (xa, wd.float(), 72), (E.Act(xa.buf.float(), 1, 1, 24, 64), wd, 72), (E.Act(xa.buf.float(), 1, 1, 24, 64), wd.float(), 72), (xa, wd[0], 72)):
        with pytest.raises(L.SdmiError):
            E.lora_gemm(x2, w2, n, **good)
    for bad in ((a.float(), b, scale), (a, b[:2], scale), (a, b, scale[:2]), (a[:, :12], b, scale), (a, b, scale.double())):
        with pytest.raises(L.SdmiError):
            E.LoraPack(*bad)


def test_lora_last_id_covers_fewer_rows():
    x, w, a, b, scale, _, _ = _lora_case(4, 150, 64, 72, 1, 16, 3, False, False)
    ids = [2, 0, 1]                                         # 64 + 64 + 22 rows
    xd, wd, ad, bd, sd, idd = x.to(DEV), w.to(DEV), a.to(DEV), b.to(DEV), scale.to(DEV), _i32(ids)
    out = torch.full((152, 80), 5.0, dtype=H16, device=DEV)
    ws = torch.empty((max(L.load().sdmi_lora_gemm_ws_bytes(150, 72, 64, 16, 1, 64), 2) // 2,), dtype=H16, device=DEV)
    L.call("sdmi_lora_gemm", xd.data_ptr(), 64, wd.data_ptr(), 64, out.data_ptr(), 80, 150, 72, 64, 0, 0, 0, ad.data_ptr(), bd.data_ptr(), sd.data_ptr(), 3, 16, 1,
           idd.data_ptr(), 64, 0, ws.data_ptr(), 2 * ws.numel(), torch.cuda.current_stream().cuda_stream)
    want, tol = _lora_oracle(x, w, a, b, scale, ids, 64, 1, None, None)
    _close(out[:150, :72], want, tol, "lora, ragged last request")
    assert bool((out[150:] == 5.0).all()) and bool((out[:, 72:] == 5.0).all())


def test_lora_residual_in_place():
    x, w, a, b, scale, bi, res = _lora_case(6, 200, 128, 136, 1, 8, 2, True, True)
    want, tol = _lora_oracle(x, w, a, b, scale, [1, 0], 100, 1, bi, res)
    stream = E.Act(res.to(DEV).view(1, 200, 136), 1, 1, 200, 136)
    E.lora_gemm(E.Act(x.to(DEV).view(1, 200, 128), 1, 1, 200, 128), w.to(DEV), 136, E.LoraPack(a.to(DEV), b.to(DEV), scale.to(DEV)), _i32([1, 0]), bias=bi.to(DEV),
                residual=stream, out=stream)
    _close(stream.buf[0], want, tol, "lora, residual in place")


@pytest.mark.skipif(H16 is torch.bfloat16, reason="bf16 does not saturate")
@pytest.mark.parametrize("per,ids,groups,rank", [(1, [0, 1, -1], 1, 8), (1, [i % 3 - 1 for i in range(40)], 2, 16), (80, [1, 0], 3, 8), (80, [1, 0], 1, 64), (1, [i % 3 - 1 for i in range(160)], 1, 24)])
def test_range_audit_sees_a_clipped_low_rank_factor(per, ids, groups, rank):
    """x a^T past the 16-bit range while the result, through a small b, is well inside: reported, with how many of it."""
    m, k, n = per * len(ids), 128, 48 * groups
    x, w, a, b, scale, _, _ = _lora_case(1, m, k, n, groups, rank, 2, False, False)
    x, b, scale = x.abs() + 1.0, b * 2.0 ** -14, torch.tensor([1.0, 500.0])
    a = a.abs()
    a[1, 3] = 8.0                                               # adapter 1, rank 3: a sum past 1024, times 500
    want = sum(per for j in ids if j == 1)
    E.RANGE_LOG.clear()
    E.RANGE_AUDIT = True
    try:
        y = _run_lora(x, w, a, b, scale, ids, None, None)
        assert torch.isfinite(y).all()
        rows = [e for e in E.RANGE_LOG if "low-rank" in e[0]]
        assert len(rows) == len(E.RANGE_LOG) == (1 if want else 0), E.RANGE_LOG
        assert all(e[1:] == (m, groups * rank, want) for e in rows), E.RANGE_LOG
        assert E.RANGE_AUDIT
    finally:
        E.RANGE_AUDIT = False
        E.RANGE_LOG.clear()


# ------------------------------------------------------------------------------------------------------------ streams and graphs
def _both(seed, nq, nkv):
    """A projection with adapters whose result attends to encoder states, as a block of the UNet does; returns a function that runs it."""
    rs = np.random.RandomState(seed)
    x, w, a, b, scale, _, _ = _lora_case(seed, 2 * nq, 128, 128, 1, 16, 3, False, False)
    kv = _h(rs, 2, nkv, 256).to(DEV)
    lens, index, ids = _i32([nkv, nkv // 2]), _i32([0, 1]), _i32([0, 1])
    xa, wd, pack = E.Act(x.to(DEV).view(2, nq, 128), 2, 1, nq, 128), w.to(DEV), E.LoraPack(a.to(DEV), b.to(DEV), scale.to(DEV))
    kva = E.Act(kv, 2, 1, nkv, 256)

    def run():
        q = E.lora_gemm(xa, wd, 128, pack, ids)
        return E.cross_attention(q, kva.cols(0, 128), kva.cols(128, 128), 2, index=index, lens=lens).buf
    return run, lens, index, ids


@pytest.mark.parametrize("nq,nkv", [(1, 2000), (144, 77)])
def test_two_streams_at_once_give_the_bits_of_one(nq, nkv):
    runs = [_both(s, nq, nkv)[0] for s in (1, 2)]
    alone = [r().clone() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(runs[i]())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


@pytest.mark.parametrize("nq,nkv", [(1, 2000), (144, 77)])
def test_graphs_replayed_together_see_new_lengths_and_ids(nq, nkv):
    """Two captured graphs replayed on two streams at once; lengths, contexts and adapters change between the replays."""
    made = [_both(s, nq, nkv) for s in (3, 4)]
    graphs, outs = [], []
    for run, _, _, _ in made:
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        want = []
        for run, lens, index, ids in made:
            lens.copy_(_i32([nkv - step, 1 + 17 * step]))
            index.copy_(_i32([step % 2, 1]))
            ids.copy_(_i32([step - 1, 2]))
            want.append(run().clone())                  # eager work between the replays
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), step
