"""K / V pages of 16-bit numbers: attention against float64 on the same numbers.

Bounds, per output number, with u = eps / 2 of the type (2^-8 bf16, 2^-11 fp16):
  score   d = (128 + 8) 2^-24 scale sum |q| |k| + 2^-21 (|S before the bias| + |bias|)
          (fp32 products and sums, the cap's function to a few steps, the bias' product
          and sum);
  output  probabilities may be rounded to the type once and the output is, and fp16
          probabilities below 2^-31 of the largest vanish:
          |out - ref| <= u (|ref| + A) (1 + u) + 2 d A + [fp16] n 2^-31 max |v|,  A = sum_j p_j |v_j|;
  lse     |lse - ref| <= d + 2^-21 (1 + |ref|)."""
import math

import pytest
import torch

from conftest import pkg

PG = pkg("paged")
DEV = "cuda:0"
gpu = pytest.mark.gpu
BF16, F16, I32 = torch.bfloat16, torch.float16, torch.int32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(g, lens, kv_heads, dtype, major="token", spare=3, fill=math.nan):
    """Pools whose rows behind each request's length, and whose unused pages, hold `fill`, and the table (-1 behind
    each request's pages)."""
    need = [-(-n // 64) for n in lens]
    pages, width = sum(need) + spare, max(need + [1]) + 2
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    table = torch.full((len(lens), width), -1, dtype=I32)
    shape = (pages, 64, kv_heads, 128) if major == "token" else (pages, kv_heads, 64, 128)
    pools = []
    for _ in range(2):
        pool = torch.full(shape, fill, device=DEV, dtype=dtype)
        pools.append(pool if major == "token" else pool.transpose(1, 2))
    at = 0
    for r, n in enumerate(lens):
        for e in range(need[r]):
            table[r, e] = order[at]
            rows = min(64, n - 64 * e)
            for pool in pools:
                pool[order[at], :rows] = torch.randn((rows, kv_heads, 128), generator=g, device=DEV).to(dtype)
            at += 1
    return pools, table.to(DEV)


def chains(parents):
    out = []
    for i in range(len(parents)):
        path = [i]
        while 0 <= parents[path[-1]] < path[-1]:
            path.append(parents[path[-1]])
        out.append(path)
    return out


def seen_and_distance(nq, n, window=0, prefix=0, document=None, parents=None):
    """[nq, n] whether query i sees key j, and |position - position of j|."""
    j, i = torch.arange(n), torch.arange(nq)
    if parents is None:
        pos = n - nq + i[:, None]
        first = torch.zeros((nq, 1), dtype=torch.long) if document is None else document.cpu().long()[:, None]
        if window:
            first = torch.maximum(first, pos - window + 1)
        return (((j <= pos) & (j >= first)) | (j < prefix)).to(DEV), (pos - j).abs().to(DEV)
    before, seen, away = n - nq, torch.zeros((nq, n), dtype=torch.bool), torch.zeros((nq, n), dtype=torch.long)
    for q, path in enumerate(chains(parents)):
        pos = before + len(path) - 1
        for k in range(max(before, 0)):
            seen[q, k] = not window or k >= pos - window + 1
            away[q, k] = abs(pos - k)
        for step, a in enumerate(path):
            if before + a >= 0:
                seen[q, before + a] = True
                away[q, before + a] = step
    return seen.to(DEV), away.to(DEV)


def reference(q, k, v, seen, away, scale, cap=0.0, slopes=None):
    """q [nq, heads, 128], k, v [n, kv_heads, 128] -> out, A, lse, d, max |v| in float64."""
    nq, heads, _ = q.shape
    group = heads // k.shape[1]
    out, mag, lse, d, most = [], [], [], [], []
    for h in range(heads):
        kh, vh, qh = k[:, h // group].double(), v[:, h // group].double(), q[:, h].double()
        visible = seen.any(0)
        kh, vh = kh.masked_fill(~visible[:, None], 0.0), vh.masked_fill(~visible[:, None], 0.0)
        s = scale * (qh @ kh.T)
        err = (128 + 8) * 2.0 ** -24 * scale * (qh.abs() @ kh.abs().T)
        if cap:
            s = cap * torch.tanh(s / cap)
        err = err + 2.0 ** -21 * s.abs()
        if slopes is not None:
            bias = slopes[h].double() * away
            s, err = s - bias, err + 2.0 ** -21 * bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        l = torch.logsumexp(s, 1)
        p = torch.exp(s - l[:, None]).masked_fill(~seen, 0.0)
        out.append(p @ vh), mag.append(p @ vh.abs()), lse.append(l)
        d.append(err.masked_fill(~seen, 0.0).amax(1) if k.shape[0] else l * 0)
        most.append(vh.abs().amax() if k.shape[0] else l.sum() * 0)
    return torch.stack(out, 1), torch.stack(mag, 1), torch.stack(lse, 1), torch.stack(d, 1), torch.stack(most)


def rows_of(pool, table, n):
    at = torch.arange(n, device=DEV)
    return pool[table[at // 64].long(), at % 64]


def check(out, lse, q, k, v, seen, away, scale=128 ** -0.5, cap=0.0, slopes=None):
    u = torch.finfo(out.dtype).eps / 2
    ref, mag, ref_lse, d, most = reference(q, k, v, seen, away, scale, cap, slopes)
    none = ~seen.any(1)
    if bool(none.any()):
        assert bool((out[none] == 0).all()) and bool((lse[none] == -math.inf).all())
    some = ~none
    tiny = k.shape[0] * 2.0 ** -31 * most[None, :, None] if out.dtype == F16 else 0.0
    bound = (u * (ref.abs() + mag) * (1 + u) + 2 * d[..., None] * mag + tiny)[some] + 1e-30
    off = (out.double() - ref).abs()[some]
    assert bool((off <= bound).all()), float((off / bound).max())
    off = ((lse.double() - ref_lse).abs() / (d + 2.0 ** -21 * (1 + ref_lse.abs())))[some]
    assert bool((off <= 1).all()), float(off.max())


def offsets(counts):
    return torch.tensor([0, *torch.tensor(counts, dtype=torch.long).cumsum(0).tolist()], dtype=I32, device=DEV)


def run_and_check(g, nq, lens, kv_heads, group, dtype, major="token", tree=None, prefix=None, document=None, slopes=False, cap=0.0, window=0,
                  max_q="given", scale=None, single=False):
    (kp, vp), table = make(g, lens, kv_heads, dtype, major)
    tokens, heads = sum(nq), kv_heads * group
    q = torch.randn((tokens, heads, 128), generator=g, device=DEV).mul_(1.5).to(dtype)
    cu, of_lens = offsets(nq), torch.tensor(lens, dtype=I32, device=DEV)
    sl = torch.exp2(-torch.arange(1, heads + 1, device=DEV) * 8.0 / heads).float() if slopes else None
    more = dict(softmax_scale=scale, softcap=cap, slopes=sl, window=window, return_lse=True)
    most = {"given": max(nq + [0]), None: None}[max_q]
    if tree is not None:
        out, lse = PG.attend_tree(q, kp, vp, table, of_lens, torch.tensor(sum(tree, []), dtype=I32, device=DEV), cu, most, **more)
    else:
        pre = None if prefix is None else torch.tensor(prefix, dtype=I32, device=DEV)
        doc = None if document is None else torch.cat(document).to(I32).to(DEV)
        if single:
            out, lse = PG.attend(q, kp, vp, table, of_lens, prefix=pre, document=doc, **more)
        else:
            out, lse = PG.attend(q, kp, vp, table, of_lens, cu, most, prefix=pre, document=doc, **more)
    at = 0
    for r, n in enumerate(nq):
        seen, away = seen_and_distance(n, lens[r], window, 0 if prefix is None else prefix[r], None if document is None else document[r],
                                       None if tree is None else tree[r])
        mine = slice(at, at + n)
        if n:
            check(out[mine], lse[mine], q[mine], rows_of(kp, table[r], lens[r]), rows_of(vp, table[r], lens[r]), seen, away,
                  128 ** -0.5 if scale is None else scale, cap, sl)
        at += n


# ------------------------------------------------------------------ sequences
@gpu
@pytest.mark.parametrize("lens,kv_heads,group", [([1], 1, 1), ([64, 0, 65], 1, 4), ([130, 1], 2, 8), ([300, 63, 2, 128, 129], 4, 7),
                                                 ([2000, 5], 8, 1), ([700], 3, 5), ([5000, 10, 900], 1, 16), ([200, 64], 2, 33), ([1000], 1, 71)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_single_tokens(lens, kv_heads, group, dtype):
    print("single", lens, kv_heads, group, dtype, flush=True)
    run_and_check(gen(sum(lens) + group), [1] * len(lens), lens, kv_heads, group, dtype, single=True)


@gpu
@pytest.mark.parametrize("nq,lens", [([1, 2], [1, 2]), ([65, 1, 0, 30], [65, 1, 5, 100]), ([64, 128], [128, 128]), ([3, 17, 40], [1000, 17, 63]),
                                     ([200, 1, 90], [700, 400, 91]), ([5, 0], [2, 0])])
@pytest.mark.parametrize("kv_heads,group,dtype,major", [(1, 1, BF16, "token"), (2, 4, F16, "head"), (1, 3, BF16, "head"), (4, 8, BF16, "token")])
def test_ragged_queries(nq, lens, kv_heads, group, dtype, major):
    print("ragged", nq, lens, kv_heads, group, dtype, major, flush=True)
    for max_q in ("given", None):
        run_and_check(gen(sum(lens) + group), nq, lens, kv_heads, group, dtype, major, max_q=max_q)


@gpu
@pytest.mark.parametrize("more", [dict(cap=50.0), dict(cap=1.0), dict(cap=0.1, scale=0.5), dict(slopes=True), dict(cap=5.0, slopes=True),
                                  dict(window=1), dict(window=64), dict(window=100, prefix=[3, 70, 0]), dict(prefix=[1000, 64, 33]),
                                  dict(window=37, slopes=True, cap=30.0, prefix=[1, 2, 150])])
@pytest.mark.parametrize("nq,kv_heads,group,dtype", [([1, 1, 1], 2, 4, BF16), ([80, 7, 90], 1, 3, F16), ([4, 8, 2], 4, 2, BF16),
                                                     ([150, 200, 90], 2, 6, BF16)])
def test_masks_and_scores(more, nq, kv_heads, group, dtype):
    print("masks", more, nq, kv_heads, group, dtype, flush=True)
    run_and_check(gen(kv_heads + group), nq, [500, 200, 90], kv_heads, group, dtype, **more)


@gpu
@pytest.mark.parametrize("window,prefix", [(0, None), (50, None), (0, [40, 0, 200])])
@pytest.mark.parametrize("kv_heads,group,dtype", [(1, 4, BF16), (2, 1, F16)])
def test_documents(window, prefix, kv_heads, group, dtype):
    print("documents", window, prefix, kv_heads, group, dtype, flush=True)
    nq, lens = [300, 1, 130], [300, 90, 200]
    document = []
    for n, m in zip(nq, lens):
        pos = torch.arange(m - n, m)
        document.append(pos // 37 * 37)
    document[2][5] = 10000  # (a query whose document begins behind it sees nothing but the prefix)
    document[2][6] = -7
    run_and_check(gen(7), nq, lens, kv_heads, group, dtype, document=document, window=window, prefix=prefix)


# ---------------------------------------------------------------------- trees
def random_tree(n, seed, roots=1):
    r = torch.Generator().manual_seed(seed)
    return [-1 if i < roots else int(torch.randint(0, i, (1,), generator=r)) for i in range(n)]


@gpu
@pytest.mark.parametrize("drafts,before", [([1, 2], [0, 63]), ([16, 7, 0, 64], [100, 64, 20, 1]), ([5, 33], [1000, 31]), ([100, 65], [200, 0]),
                                           ([256, 3], [70, 4000])])
@pytest.mark.parametrize("kv_heads,group,dtype", [(1, 4, BF16), (4, 1, F16), (2, 9, BF16)])
def test_trees(drafts, before, kv_heads, group, dtype):
    print("tree", drafts, before, kv_heads, group, dtype, flush=True)
    tree = [random_tree(n, n + b, 1 + b % 2) for n, b in zip(drafts, before)]
    for more in ({}, dict(cap=3.0), dict(slopes=True), dict(window=20), dict(window=70, slopes=True, cap=40.0)):
        run_and_check(gen(sum(drafts)), drafts, [a + b for a, b in zip(drafts, before)], kv_heads, group, dtype, tree=tree, **more)


@gpu
def test_parents_that_are_none():
    """Its own number, a later one and numbers below zero make a draft follow the context; chains and stars."""
    for tree in ([-1, 1, 5, 2, -9, 4, 3], list(range(-1, 40)), [-1] + [0] * 60):
        run_and_check(gen(3), [len(tree)], [len(tree) + 90], 2, 2, BF16, tree=[tree], slopes=True)
        run_and_check(gen(3), [len(tree)], [len(tree) - 2], 2, 2, BF16, tree=[tree])  # (more drafts than keys)


# --------------------------------------------------- pages and values that are out of order
@gpu
@pytest.mark.parametrize("nq,group", [(1, 4), (40, 2), (200, 2)])
def test_pages_that_are_not_there(nq, group):
    """Keys of pages below zero and past the pool are left out."""
    g = gen(11)
    lens = [700, 300]
    (kp, vp), table = make(g, lens, 1, BF16)
    table[0, 2], table[0, 7], table[1, 0] = -1, kp.shape[0], 1 << 30
    q = torch.randn((2 * nq, group, 128), generator=g, device=DEV).to(BF16)
    cu = offsets([nq, nq])
    out, lse = PG.attend(q, kp, vp, table, torch.tensor(lens, dtype=I32, device=DEV), cu, nq, return_lse=True)
    for r, n in enumerate(lens):
        seen, away = seen_and_distance(nq, n)
        ok = (table[r, torch.arange(n, device=DEV) // 64] >= 0) & (table[r, torch.arange(n, device=DEV) // 64] < kp.shape[0])
        clean = table[r].clamp(0, kp.shape[0] - 1)
        check(out[r * nq:(r + 1) * nq], lse[r * nq:(r + 1) * nq], q[r * nq:(r + 1) * nq], rows_of(kp, clean, n), rows_of(vp, clean, n),
              seen & ok, away)


@gpu
@pytest.mark.parametrize("nq,group,dtype", [(1, 4, BF16), (30, 2, F16), (150, 2, BF16)])
@pytest.mark.parametrize("odd", [math.inf, -math.inf, math.nan])
def test_odd_values_reach_those_that_see_them(nq, group, dtype, odd):
    """An infinite or NaN value of a key: the queries before it are as if it were zero."""
    print("odd", nq, group, dtype, odd, flush=True)
    g = gen(5)
    n = 200
    (kp, vp), table = make(g, [n], 1, dtype)
    q = torch.randn((nq, group, 128), generator=g, device=DEV).to(dtype)
    lens, cu = torch.tensor([n], dtype=I32, device=DEV), offsets([nq])
    at = n - 1 - nq // 2
    page, row = int(table[0, at // 64]), at % 64
    want, _ = PG.attend(q, kp, vp, table, lens, cu, nq, return_lse=True)
    vp[page, row, 0, 5] = odd
    vp[page, row, 0, 77] = -odd
    got, lse = PG.attend(q, kp, vp, table, lens, cu, nq, return_lse=True)
    sees = torch.arange(n - nq, n, device=DEV) >= at
    assert torch.equal(got[~sees], want[~sees]) and bool(torch.isfinite(lse).all())
    expect = torch.tensor(odd, device=DEV)
    for col, x in ((5, expect), (77, -expect)):
        assert bool((torch.isnan(got[sees][..., col]) if math.isnan(odd) else got[sees][..., col] == x).all())
    keep = [c for c in range(128) if c not in (5, 77)]
    assert bool(torch.isfinite(got[sees][..., keep]).all())
    # a key that scores NaN
    vp[page, row, 0, 5] = vp[page, row, 0, 77] = 1.0
    kp[page, row, 0, 3] = math.nan
    got, lse = PG.attend(q, kp, vp, table, lens, cu, nq, softcap=10.0, return_lse=True)
    assert bool(torch.isnan(got[sees]).all()) and bool(torch.isnan(lse[sees]).all())
    assert bool(torch.isfinite(got[~sees]).all()) and bool(torch.isfinite(lse[~sees]).all())


@gpu
def test_keys_that_all_score_minus_infinity():
    (kp, vp), table = make(gen(6), [70, 70], 1, BF16)
    q = torch.ones((2, 2, 128), device=DEV, dtype=BF16)
    kp[table[0, :2].long()] = -math.inf
    out, lse = PG.attend(q, kp, vp, table, torch.tensor([70, 0], dtype=I32, device=DEV), return_lse=True)
    assert bool(torch.isnan(out[0]).all()) and bool((lse == -math.inf).all()) and bool((out[1] == 0).all())


@gpu
def test_lengths_past_the_table_and_below_zero():
    (kp, vp), table = make(gen(8), [640, 640, 640], 1, BF16)
    q = torch.randn((3, 2, 128), generator=gen(9), device=DEV).to(BF16)
    lens = torch.tensor([1 << 30, -5, 100], dtype=I32, device=DEV)
    table = table[:, :10].contiguous()
    out, lse = PG.attend(q, kp, vp, table, lens, return_lse=True)
    for r, n in enumerate((640, 0, 100)):
        seen, away = seen_and_distance(1, n)
        check(out[r:r + 1], lse[r:r + 1], q[r:r + 1], rows_of(kp, table[r], n), rows_of(vp, table[r], n), seen, away)


@gpu
@pytest.mark.parametrize("group,nq", [(4, 20), (2, 300)])
def test_rows_that_are_left_alone(group, nq):
    """Rows before the first request, behind the last and past a request's first max_q."""
    g = gen(10)
    lens = [nq + 100, 60]
    (kp, vp), table = make(g, lens, 2, BF16)
    tokens = 7 + nq + 50 + 9
    cu = torch.tensor([7, 7 + nq, 7 + nq + 50], dtype=I32, device=DEV)
    q = torch.randn((tokens, 2 * group, 128), generator=g, device=DEV).to(BF16)
    q[:7] = math.nan
    q[-9:] = math.nan
    out = torch.full_like(q, 123.0)
    of_lens = torch.tensor(lens, dtype=I32, device=DEV)
    PG.attend(q, kp, vp, table, of_lens, cu, out=out)
    full = out.clone()
    assert bool((out[:7] == 123).all()) and bool((out[-9:] == 123).all()) and not bool((out[7:-9] == 123).all(-1).any())
    out.fill_(123.0)
    most = nq - 3
    PG.attend(q, kp, vp, table, of_lens, cu, most, out=out)
    assert bool((out[7 + most:7 + nq] == 123).all()) and bool((out[-9:] == 123).all())
    assert float((out[7:7 + most].float() - full[7:7 + most].float()).abs().max()) <= 2.0 ** -6


@gpu
def test_strided_tensors():
    g = gen(12)
    lens, nq = [150, 80], [20, 3]
    (kp, vp), table = make(g, lens, 2, F16)
    kw, vw = (torch.full((kp.shape[0], 66, 3, 136), math.nan, device=DEV, dtype=F16) for _ in range(2))
    kw[:, 1:65, :2, :128], vw[:, 1:65, :2, :128] = kp, vp
    q = torch.randn((23, 5, 256), generator=g, device=DEV).to(F16)[:, :4, 128:]
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=I32, device=DEV)
    wide[:, :table.shape[1]] = table
    of_lens, cu = torch.tensor(lens, dtype=I32, device=DEV), offsets(nq)
    out = torch.zeros((23, 6, 160), device=DEV, dtype=F16)[:, 1:5, 16:144]
    PG.attend(q, kw[:, 1:65, :2, :128], vw[:, 1:65, :2, :128], wide[:, :table.shape[1]], of_lens, cu, 20, out=out)
    assert torch.equal(out, PG.attend(q.contiguous(), kp, vp, table, of_lens, cu, 20))


@gpu
def test_many_requests():
    """More requests than the plan by lengths takes, and more than a wave looks at in one go."""
    g = gen(13)
    lens = [(37 * i) % 200 for i in range(300)]
    run_and_check(g, [1] * 300, lens, 1, 2, BF16, single=True)
    run_and_check(g, [min(n, i % 3) for i, n in enumerate(lens)], lens, 1, 2, BF16)
    run_and_check(g, [i % 5 * 40 if i % 50 == 0 else 1 for i in range(300)], [250] * 300, 1, 2, BF16)


@gpu
def test_empty_calls():
    (kp, vp), table = make(gen(1), [64], 1, BF16)
    lens = torch.tensor([64], dtype=I32, device=DEV)
    q = torch.randn((1, 2, 128), device=DEV).to(BF16)
    assert PG.attend(q[:0], kp, vp, table[:0], lens[:0]).shape == (0, 2, 128)
    assert PG.attend(q[:0], kp, vp, table, lens, offsets([0])).shape == (0, 2, 128)
    for pools, t in (((kp[:0], vp[:0]), table), ((kp, vp), table[:, :0])):
        out, lse = PG.attend(q, *pools, t, lens, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
