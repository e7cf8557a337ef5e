"""Attention over keys and values expanded from the latent, ragged sequences,
against float64.

Bounds, per output number, with u = 2^-8 (bf16's half step relative to the value):
probabilities and output are each rounded to bf16 once, scores and sums are fp32:
with d = (192 + 8) 2^-24 scale sum |q| |k| + 2^-21 |score|,
  |out - ref| <= u (|ref| + A) (1 + u) + 2 d A,  A = sum_j p_j |v_j|,
  |lse - ref| <= d + 2^-21 (1 + |ref|)."""
import importlib
import math

import pytest
import torch

from conftest import pkg

LT = pkg("latent")
DEV = "cuda:0"
U = 2.0 ** -8
gpu = pytest.mark.gpu


def inputs(seed, nq, nk, heads, amp=1.5, behind=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, device=DEV, generator=g)
    q = (amp * r(sum(nq) + behind, heads, 192)).to(torch.bfloat16)
    kv = r(sum(nk) + behind, heads, 256).to(torch.bfloat16)
    rope = r(sum(nk) + behind, 64).to(torch.bfloat16)
    cu = lambda n: torch.tensor([0] + n, device=DEV).cumsum(0).to(torch.int32)
    return q, kv, rope, cu(nq), cu(nk)


def check(out, lse, q, kv, rope, nq, nk, causal=True, scale=192 ** -0.5):
    a = b = 0
    for n, m in zip(nq, nk):
        qq, kk, vv = q[a:a + n].double(), kv[b:b + m, :, :128].double(), kv[b:b + m, :, 128:].double()
        kk = torch.cat([kk, rope[b:b + m].double()[:, None].expand(-1, q.shape[1], -1)], 2)
        i = torch.arange(n, device=DEV)[:, None]
        seen = torch.arange(m, device=DEV)[None] <= (m - n + i if causal else i * 0 + m)
        for h in range(q.shape[1]):
            o, l = out[a:a + n, h].double(), lse[a:a + n, h].double()
            s = scale * (qq[:, h] @ kk[:, h].T)
            d = (((192 + 8) * 2.0 ** -24 * scale) * (qq[:, h].abs() @ kk[:, h].abs().T) + 2.0 ** -21 * s.abs())
            s = s.masked_fill(~seen, -math.inf)
            some = seen.any(1)
            assert bool((o[~some] == 0).all()) and bool((l[~some] == -math.inf).all())
            if not bool(some.any()):
                continue
            o, l, s, d = o[some], l[some], s[some], d.masked_fill(~seen, 0.0).amax(1)[some]
            ref_l = torch.logsumexp(s, 1)
            p = torch.exp(s - ref_l[:, None])
            ref, mag = p @ vv[:, h], p @ vv[:, h].abs()
            bound = U * (ref.abs() + mag) * (1 + U) + 2 * d[:, None] * mag
            off = (o - ref).abs()
            assert bool((off <= bound).all()), (n, m, h, float((off / bound).max()))
            off = (l - ref_l).abs() / (d + 2.0 ** -21 * (1 + ref_l.abs()))
            assert bool((off <= 1).all()), (n, m, h, float(off.max()))
        a, b = a + n, b + m


@gpu
@pytest.mark.parametrize("nq,nk,heads", [
    ([1], [1], 1), ([1], [700], 2), ([64], [64], 1), ([65], [65], 3), ([33, 1, 0, 127, 200], None, 2),
    ([5, 300], [70, 1000], 2), ([128], [128], 16), ([257], [1500], 1), ([100, 7], [50, 7], 2), ([40], [0], 1),
    ([2, 3, 4], [9000, 30, 4], 1), ([1300, 900], None, 16), ([8, 8, 8, 8], [512, 512, 512, 512], 16),
    ([3, 2100, 5, 1, 0, 2, 64, 300, 1, 1, 9, 4, 700], None, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences(nq, nk, heads, causal):
    print("expanded", nq, nk, heads, causal, flush=True)
    nk = nq if nk is None else nk
    q, kv, rope, cu_q, cu_k = inputs(sum(nq) + heads, nq, nk, heads)
    out, lse = LT.attend_expanded(q, kv, rope, cu_q, None if nk is nq else cu_k, max(nq), causal=causal, return_lse=True)
    check(out, lse, q, kv, rope, nq, nk, causal)


@gpu
def test_work_groups_of_256_queries():
    """Enough queries and heads that every CU has 256 of them."""
    print("expanded wide", flush=True)
    nq, nk = [700, 4300], [1100, 4300]
    q, kv, rope, cu_q, cu_k = inputs(9, nq, nk, 16)
    out, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max(nq), return_lse=True)
    check(out[:, ::5], lse[:, ::5], q[:, ::5], kv[:, ::5], rope, nq, nk)


@gpu
def test_strides_and_rows_behind_the_last_sequence():
    print("expanded strides", flush=True)
    nq, nk = [70, 20], [200, 90]
    q, kv, rope, cu_q, cu_k = inputs(5, nq, nk, 3, amp=6.0, behind=40)
    wide = torch.zeros((q.shape[0], 4, 200), device=DEV, dtype=torch.bfloat16)
    wide[:, 1:, 8:] = q
    both = torch.zeros((kv.shape[0], 3 * 256 + 64 + 16), device=DEV, dtype=torch.bfloat16)
    both[:, :768], both[:, 768:832] = kv.reshape(-1, 768), rope
    both[sum(nk):] = math.nan  # behind the last key
    wide[sum(nq):] = math.nan
    space = torch.full((q.shape[0], 3, 136), 7.0, device=DEV, dtype=torch.bfloat16)
    args = wide[:, 1:, 8:], both[:, :768].unflatten(1, (3, 256)), both[:, 768:832], cu_q, cu_k
    out, lse = LT.attend_expanded(*args, 70, softmax_scale=0.1, out=space[..., 4:132], return_lse=True)
    check(out, lse, q, kv, rope, nq, nk, scale=0.1)
    assert bool((space[..., :4] == 7).all()) and bool((space[..., 132:] == 7).all()) and bool((space[90:] == 7).all())
    # without max_q, and in parts of the keys (one sequence, one head, few queries)
    assert torch.equal(LT.attend_expanded(*args, softmax_scale=0.1)[:90], out[:90])
    space.fill_(7.0)
    cu_q, cu_k = (torch.tensor(x, device=DEV, dtype=torch.int32) for x in ([3, 9], [0, 290]))
    both[sum(nk):] = 0.5
    out, lse = LT.attend_expanded(wide[:, 1:2, 8:], both[:, :256].unflatten(1, (1, 256)), both[:, 768:832], cu_q, cu_k, 6,
                                  out=space[:, :1, 4:132], return_lse=True)
    check(out[3:9], lse[3:9], q[3:9, :1], kv[:, :1], rope, [6], [290])
    assert bool((space[:3] == 7).all()) and bool((space[9:] == 7).all())


@gpu
@pytest.mark.parametrize("heads,n", [(1, 300), (16, 2100), (1, 2100)])
def test_values_that_are_not_finite(heads, n):
    """An infinite or NaN value, or key, of a token that a query does not see changes
    nothing for that query; those that see it get what the formula gives."""
    print("expanded special", heads, n, flush=True)
    q, kv, rope, cu, _ = inputs(3, [n], [n], heads, amp=0.2)
    clean, _ = LT.attend_expanded(q, kv, rope, cu, None, n, return_lse=True)
    bad = kv.clone()
    h = heads - 1
    bad[100, h, 130], bad[110, h, 131], bad[120, h, 132], bad[170, h, 132] = math.inf, -math.inf, math.inf, -math.inf
    bad[200, h, 140] = math.nan
    bad[250, h, 3] = math.nan  # a key
    out, lse = LT.attend_expanded(q, bad, rope, cu, None, n, return_lse=True)
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[:, :h], clean[:, :h])
    o, c = out[:250, h].float(), clean[:250, h].float()
    assert bool((o[100:, 2] == math.inf).all()) and bool((o[110:, 3] == -math.inf).all())
    assert bool((o[120:170, 4] == math.inf).all()) and bool(o[170:, 4].isnan().all()) and bool(o[200:, 12].isnan().all())
    rest = [i for i in range(128) if i not in (2, 3, 4, 12)]
    assert torch.equal(o[:, rest], c[:, rest])
    assert torch.equal(o[:100, 2], c[:100, 2]) and torch.equal(o[:110, 3], c[:110, 3]) and torch.equal(o[:200, 12], c[:200, 12])
    assert bool(out[250:, h].isnan().all()) and bool(lse[250:, h].isnan().all()) and not bool(lse[:250].isnan().any())


@gpu
def test_rows_past_32_bits():
    """Queries, keys, rope keys and outputs whose last rows lie 2^32 numbers behind the first."""
    print("expanded far rows", flush=True)
    n, heads, row = 300, 2, 1 << 24
    q, kv, rope, cu, _ = inputs(11, [n], [n], heads)
    base = torch.empty(n * row, device=DEV, dtype=torch.bfloat16)
    far = lambda t, at: base.as_strided((n, *t.shape[1:]), (row, *t.stride()[1:]), at).copy_(t)
    fq, fkv, frope = far(q, 0), far(kv, 8192), far(rope, 16384)
    out = base.as_strided((n, heads, 128), (row, 128, 1), 32768).fill_(7)
    _, lse = LT.attend_expanded(fq, fkv, frope, cu, out=out, return_lse=True)
    check(out, lse, q, kv, rope, [n], [n])
    whole, whole_lse = LT.attend_expanded(q, kv, rope, cu, return_lse=True)
    assert torch.equal(out, whole) and torch.equal(lse, whole_lse)


@gpu
def test_lengths_outside_the_tensors():
    """cu_q and cu_k past the tensors or descending are clamped."""
    print("expanded clamped", flush=True)
    q, kv, rope, _, _ = inputs(6, [50], [80], 2)
    cu = lambda *x: torch.tensor(x, device=DEV, dtype=torch.int32)
    out = LT.attend_expanded(q, kv, rope, cu(0, 1000), cu(0, 1 << 30), 1000)
    assert torch.equal(out, LT.attend_expanded(q, kv, rope, cu(0, 50), cu(0, 80), 50))
    keep = torch.full_like(out, 3.0)
    LT.attend_expanded(q, kv, rope, cu(20, 10), cu(-5, -9), 50, out=keep)
    assert bool((keep == 3).all())


@gpu
def test_absorbed_and_expanded_agree():
    """A run of the operators as a model has them: a prompt's latents attended in the
    expanded form, stored, then the same queries absorbed over the stored rows.  The
    rows hold 4 significant bits (2^-4 of each number), so the two differ by that
    order; on latents that the codes hold exactly they differ by bf16's rounding of
    the projections alone (k, q and v each 2^-8 of their magnitudes)."""
    print("expanded / absorbed", flush=True)
    g = torch.Generator(device=DEV).manual_seed(8)
    r = lambda *s: torch.randn(s, device=DEV, generator=g)
    n, heads = 200, 16
    codes = (r(n, 512) * 0.5).clamp(-3, 3).to(torch.float8_e4m3fn)
    latent, rope = codes.float().to(torch.bfloat16), r(n, 64).to(torch.bfloat16)
    w_k, w_v = (r(heads, 128, 512) / 512 ** 0.5 for _ in range(2))
    q = r(n, heads, 192).to(torch.bfloat16)
    lat = latent.float()
    kv = torch.cat([torch.einsum("hdc,nc->nhd", w_k, lat), torch.einsum("hdc,nc->nhd", w_v, lat)], 2).to(torch.bfloat16)
    cu = torch.tensor([0, n], device=DEV, dtype=torch.int32)
    out = LT.attend_expanded(q, kv, rope, cu, None, n)
    pool = torch.zeros((512, 656), device=DEV, dtype=torch.uint8)
    slots = torch.randperm(512, device=DEV, generator=g)[:n].to(torch.int32)
    LT.store_rows(latent, rope, pool, slots)
    qa = torch.cat([torch.einsum("nhd,hdc->nhc", q[..., :128].float(), w_k), q[..., 128:].float()], 2).to(torch.bfloat16)
    lens = torch.arange(1, n + 1, device=DEV, dtype=torch.int32)
    o = LT.attend(qa, pool, slots[None].expand(n, -1), lens=lens)
    back = torch.einsum("nhc,hdc->nhd", o.float(), w_v)
    # scores: rounding of k and of the absorbed q, 2^-8 of sum |q||k| each at most; values and outputs likewise
    s = 192 ** -0.5 * (torch.einsum("nhd,mhd->hnm", q[..., :128].float().abs(), kv[..., :128].float().abs()).amax((1, 2))
                       + torch.einsum("nhc,mc->hnm", qa[..., :512].float().abs(), lat.abs()).amax((1, 2)))
    bound = 2 * U * (2 * s[None, :, None] + 4) * torch.einsum("nc,hdc->hd", lat.abs().amax(0, keepdim=True), w_v.abs())[None]
    assert bool(((back - out.float()).abs() <= bound).all())
    rel = float((back - out.float()).norm() / out.float().norm())
    assert rel < 8 * U, rel


def test_refusals(monkeypatch):
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    cu = torch.zeros(2, dtype=torch.int32)
    base = dict(q=z(4, 2, 192), kv=z(5, 2, 256), k_rope=z(5, 64), cu_q=cu, cu_k=cu, max_q=4)
    with pytest.raises(ValueError, match="device"):
        LT.attend_expanded(**base)
    monkeypatch.setattr(importlib.import_module("10_20_amd._lib"), "require_gpu", lambda *t: None)
    for bad, text in ((dict(q=z(4, 2, 128)), "q must"), (dict(q=z(4, 2, 192).float()), "q must"), (dict(q=z(4, 0, 192)), "q must"),
                      (dict(kv=z(5, 3, 256)), "kv must"), (dict(kv=z(5, 2, 192)), "kv must"), (dict(k_rope=z(4, 64)), "k_rope must"),
                      (dict(cu_q=cu.long()), "cu_q must"), (dict(cu_q=cu[:0]), "cu_q must"), (dict(cu_k=cu[:1]), "cu_k must"),
                      (dict(max_q=-1), "max_q"), (dict(softmax_scale=0.0), "scale"), (dict(softmax_scale=math.nan), "scale"),
                      (dict(out=z(4, 2, 192)), "out must")):
        with pytest.raises(ValueError, match=text):
            LT.attend_expanded(**{**base, **bad})


def test_library_refusals():
    L = pkg("_lib")
    if not L.LIB_PATH.exists():
        pkg("build").build()
    h = L.lib()
    def call(fields):
        return h.v1_latent_expanded(L.PACKED["v1_latent_expanded"].pack(*fields.values()), None)

    base = dict(q=256, qr=384, qh=192, kv=256, kr=512, kh=256, rope=256, rr=64, cu_q=256, cu_k=256, out=256, o_row=256, o_head=128,
                lse=0, ws=0, wsb=0, tokens=4096, keys=4096, batch=1, heads=16, max_q=4096, causal=1, scale=0.1)
    for bad in (dict(q=8), dict(kv=8), dict(rope=4), dict(qr=380), dict(kh=252), dict(out=4), dict(o_row=254), dict(heads=0),
                dict(tokens=-1), dict(scale=0.0), dict(scale=-1.0), dict(heads=1 << 16), dict(tokens=1, max_q=1, heads=1)):
        assert call({**base, **bad}) == L.V1_ERR_INVALID, bad
        assert b"latent_expanded" in h.v1_last_error()
    for none in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert call({**base, **none}) == 0
    assert h.v1_latent_expanded(None, None) == L.V1_ERR_INVALID
