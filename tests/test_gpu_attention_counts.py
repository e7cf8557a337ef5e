"""That every key is attended once: with queries of zeros every probability is 1 / n,
so the log-sum-exp is log(n), and value numbers that are 256 in one column for each
key (column j mod the value's dims for key j) make an output of 256 / n times the
column's keys.  Sums of ones and of 256 are exact in fp32 and in bf16 products, so
that what is left is one rounding of the output (2^-8 of it), 1 / n and the
logarithm (2^-21 of 1 + log n); one key more or less moves a column by 1 / 60 or more
and exp(lse) by 1.  Lengths lie at the edges of tiles (64 keys) and of parts, rows and
heads on both sides of the rules that choose how keys are split.

And that the precision is what the kernels say: the error against 64 bits, beside
that of the exact result rounded to bf16 (e).  Probabilities that are rounded to
bf16 once add an error of the same size where the values have no mean (each term off by
as much, relative to its own magnitude, as the output is: sqrt(2) e together); two bf16
numbers leave 2^-17 of each, nothing beside e."""
import math
import random

import pytest
import torch

import test_gpu_kv8 as kv8
import test_gpu_latent as latent
from conftest import pkg

LT, K8 = pkg("latent"), pkg("kv8")
DEV = "cuda:0"
gpu = pytest.mark.gpu
BF16, I32, F8 = torch.bfloat16, torch.int32, torch.float8_e4m3fn


def counted(lse, n):
    """lse of any shape, n keys."""
    if n == 0:
        return bool((lse == -math.inf).all())
    return bool((torch.exp(lse.double()).round() == n).all())


def marked(out, columns, n):
    """out [..., dims]: columns [dims] keys of each column, n in all."""
    want = (256.0 * columns.double() / max(n, 1)).to(out.device)
    return bool(((out.double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -10) * want).all())


def columns_of(j, dims):
    return torch.bincount(j.cpu() % dims, minlength=dims)


def test_the_checks_see_one_key():
    """On the CPU: outputs as a right kernel gives them, told from those of a key more or less."""
    for dims, ns in ((512, (1, 63, 64, 65, 1000, 4097, 30000)), (128, (1, 63, 64, 65, 1000, 4097, 7680))):
        for n in ns:
            lse = torch.tensor(n).log2().float() * math.log(2)
            out = (256 * columns_of(torch.arange(n), dims) * (torch.tensor(1.0) / n)).to(BF16)
            assert counted(lse, n) and marked(out, columns_of(torch.arange(n), dims), n)
            for m in (n - 1, n + 1):
                assert not counted(lse, m)
            lost = columns_of(torch.cat([torch.arange(n // 2), torch.arange(n // 2 + 1, n)]), dims)
            twice = columns_of(torch.cat([torch.arange(n), torch.tensor([n // 2])]), dims)
            assert not marked(out, lost, n) and not marked(out, twice, n)
    assert counted(torch.tensor(-math.inf), 0) and not counted(torch.tensor(0.0), 0)


def edge_lengths(rows, most, seed):
    """Lengths around tiles' and parts' edges, the longest and none among them."""
    rng = random.Random(seed)
    edges = [most, 0, 1, 63, 64, 65, most - 1, 127, 128, 129, 255, 256, 257, 511, 513]
    edges += [min(most, max(0, 64 * rng.randint(0, most // 64) + rng.choice([-1, 0, 1]))) for _ in range(rows)]
    lens = [min(n, most) for n in edges][:rows]
    rng.shuffle(lens)
    return lens


def marked_latents(n):
    """Row j: 256 in column j % 512, codes and scales that vary by row and block, the rest zeros."""
    pool = torch.zeros((n, 656), device=DEV, dtype=torch.uint8)
    j = torch.arange(n, device=DEV)
    scale = torch.exp2(((j[:, None] // 3 + torch.arange(4, device=DEV)) % 4).float())
    codes = torch.zeros((n, 512), device=DEV)
    codes[j, j % 512] = 256.0 / scale[j, j % 512 // 128]
    pool[:, :512] = codes.to(F8).view(torch.uint8)
    pool[:, 640:] = scale.view(torch.uint8)
    return pool


@gpu
@pytest.mark.parametrize("rows,heads,most", [(1, 1, 1), (1, 16, 30000), (3, 16, 30000), (7, 64, 20000), (5, 33, 9000), (40, 16, 5000),
                                             (127, 128, 700), (128, 128, 700), (255, 16, 900), (256, 16, 900), (257, 16, 900), (300, 40, 300),
                                             (600, 64, 500)])
def test_latent_lengths(rows, heads, most):
    """Whole contexts of a page table, planned by their lengths or not; and ids of them."""
    print("count latent", rows, heads, most, flush=True)
    pool = marked_latents(-(-most // 64) * 64)
    entries = pool.shape[0] // 64
    lens = edge_lengths(rows, most, rows + heads)
    q = torch.zeros((rows, heads, 576), device=DEV, dtype=BF16)
    table = torch.arange(entries, device=DEV, dtype=I32)
    n = torch.tensor(lens, device=DEV, dtype=I32)
    columns = {m: columns_of(torch.arange(m), 512) for m in set(lens)}
    ids = torch.arange(most, device=DEV, dtype=I32).expand(rows, -1)
    for out, lse in (LT.attend(q, pool, table=table, page_bits=6, lens=n, return_lse=True), LT.attend(q, pool, ids, lens=n, return_lse=True)):
        for r, m in enumerate(lens):
            assert counted(lse[r], m), (r, m, torch.exp(lse[r].double()))
            assert marked(out[r], columns[m], m), (r, m)


@gpu
@pytest.mark.parametrize("rows,heads,keys", [(1, 16, 2048), (8, 16, 2048), (128, 16, 2047), (100, 64, 2048), (3, 32, 6000), (1, 128, 12345),
                                             (300, 16, 130), (20, 24, 63)])
def test_latent_chosen_keys(rows, heads, keys):
    """Ids in random order with holes, no lengths: rows of one capacity."""
    print("count latent ids", rows, heads, keys, flush=True)
    g = torch.Generator(device=DEV).manual_seed(keys)
    pool = marked_latents(keys + 100)
    ids = torch.stack([torch.randperm(keys + 100, device=DEV, generator=g)[:keys] for _ in range(rows)]).to(I32)
    ids[torch.rand(ids.shape, device=DEV, generator=g) < 0.1] = -1
    ids[rows // 2, keys // 2:] = -1
    ids[:, 0] = 7
    out, lse = LT.attend(torch.zeros((rows, heads, 576), device=DEV, dtype=BF16), pool, ids, return_lse=True)
    for r in range(rows):
        j = ids[r][ids[r] >= 0]
        assert counted(lse[r], j.numel()), (r, j.numel(), torch.exp(lse[r].double()))
        assert marked(out[r], columns_of(j, 512), j.numel()), r


def marked_pages(pages, heads):
    """Codes and V scales: 256 in column (position in the pool) % 128, scales by page and head."""
    at = torch.arange(pages * 64, device=DEV)
    scale = torch.exp2(((torch.arange(pages, device=DEV)[:, None] + torch.arange(heads, device=DEV)) % 4).float())
    v = torch.zeros((pages * 64, heads, 128), device=DEV)
    v[at, :, at % 128] = 256.0 / scale[at // 64]
    return v.view(pages, 64, heads, 128).to(F8), scale


@gpu
@pytest.mark.parametrize("rows,heads,group,most", [(1, 1, 1, 1), (1, 1, 4, 7680), (3, 2, 16, 7680), (6, 4, 8, 7680), (6, 8, 2, 7680), (48, 4, 8, 3000),
                                                   (40, 8, 4, 2000), (130, 3, 1, 900), (127, 16, 1, 700), (128, 16, 1, 700), (255, 8, 1, 600),
                                                   (256, 8, 1, 600), (257, 8, 4, 600), (300, 4, 4, 700), (511, 4, 1, 300), (600, 12, 1, 200)])
def test_kv8_lengths(rows, heads, group, most):
    """Whole contexts, one, two or four KV heads to a work-group, one or several sets of
    them, planned by their lengths or not; and ids of them."""
    print("count kv8", rows, heads, group, most, flush=True)
    entries = -(-most // 64)
    v, scale = marked_pages(entries, heads)
    k = torch.full(v.shape, 3.0, device=DEV).to(F8)
    lens = edge_lengths(rows, most, rows + heads)
    q = torch.zeros((rows, heads * group, 128), device=DEV, dtype=BF16)
    table = torch.arange(entries, device=DEV, dtype=I32)
    n = torch.tensor(lens, device=DEV, dtype=I32)
    columns = {m: columns_of(torch.arange(m), 128) for m in set(lens)}
    ids = torch.arange(most, device=DEV, dtype=I32).expand(rows, -1)
    for out, lse in (K8.attend(q, k, v, scale, scale, table, n, return_lse=True), K8.attend(q, k, v, scale, scale, table, n, ids, return_lse=True)):
        for r, m in enumerate(lens):
            assert counted(lse[r], m), (r, m, torch.exp(lse[r].double()))
            assert marked(out[r], columns[m], m), (r, m)


@gpu
@pytest.mark.parametrize("rows,heads,group,entries", [(6, 4, 8, 60), (6, 8, 4, 60), (40, 8, 2, 30), (130, 12, 1, 9), (255, 8, 1, 5), (256, 8, 1, 5), (300, 4, 2, 4)])
def test_kv8_contexts_of_many_heads(rows, heads, group, entries):
    """Random queries over whole contexts of 4, 8 and 12 KV heads: each head its own keys and scales."""
    print("kv8 heads", rows, heads, group, entries, flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows)
    (kp, ks), (vp, vs) = kv8.rand_pool(g, 50, heads), kv8.rand_pool(g, 50, heads, "head")
    table = torch.randint(0, 50, (rows, entries), device=DEV, generator=g, dtype=I32)
    lens = torch.tensor(edge_lengths(rows, entries * 64, rows), device=DEV, dtype=I32)
    q = torch.randn((rows, heads * group, 128), device=DEV, generator=g).to(BF16)
    out, lse = K8.attend(q, kp, vp, ks, vs, table, lens, return_lse=True)
    at = torch.arange(entries * 64, device=DEV)
    some = sorted({*range(0, rows, max(1, rows // 12)), rows - 1})
    kv8.check(out[some], lse[some], q[some], [kp, vp, ks, vs], [kv8.keys_of(table[r], at, int(lens[r]), 50) for r in some])


@gpu
@pytest.mark.parametrize("nq,nk,heads,max_q", [
    ([1], [7680], 1, 1), ([65], [7680], 2, 65), ([300], [5000], 16, 300), ([256, 257, 1], [256, 257, 1], 3, 257), ([1, 2, 3], [64, 65, 4000], 4, None),
    ([700, 20, 0, 1300], [700, 30, 0, 2000], 2, 1300), ([700, 20, 0, 1300], [700, 30, 0, 2000], 40, None), ([20] * 60 + [1100], [90] * 60 + [1100], 1, None)])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded_keys(nq, nk, heads, max_q, causal):
    print("count expanded", nq[:4], heads, causal, flush=True)
    cu = lambda n: torch.tensor([0] + n, device=DEV).cumsum(0).to(I32)
    keys = sum(nk)
    kv = torch.zeros((keys, heads, 256), device=DEV, dtype=BF16)
    j = torch.cat([torch.arange(m, device=DEV) for m in nk])
    kv[torch.arange(keys, device=DEV), :, 128 + j % 128] = 256.0
    kv[..., :128] = 1.0
    rope = torch.ones((keys, 64), device=DEV, dtype=BF16)
    q = torch.zeros((sum(nq), heads, 192), device=DEV, dtype=BF16)
    out, lse = LT.attend_expanded(q, kv, rope, cu(nq), cu(nk), max_q, causal=causal, return_lse=True)
    a = 0
    for n, m in zip(nq, nk):
        seen = torch.arange(n, device=DEV) + (m - n + 1) if causal else torch.full((n,), m, device=DEV)
        seen = seen.clamp_min(0)
        got = lse[a:a + n].double()
        assert bool((torch.exp(got).round() == seen[:, None]).all()), (n, m)
        want = 256.0 * ((seen[:, None] + 127 - torch.arange(128, device=DEV)) // 128).double() / seen.clamp_min(1)[:, None]
        off = (out[a:a + n].double() - want[:, None]).abs()
        assert bool((off <= 2.0 ** -8 * (1 + 2.0 ** -10) * want[:, None]).all()), (n, m)
        a += n


def errors(out, ref):
    """Root mean square errors of the output and of the exact result rounded to bf16."""
    rms = lambda x: float(x.double().square().mean().sqrt())
    return rms(out.double() - ref), rms(ref.to(BF16).double() - ref)


@gpu
@pytest.mark.parametrize("rows,heads,keys", [(200, 16, 300), (200, 32, 300), (4, 16, 4000), (4, 24, 9000), (300, 128, 200), (2, 64, 20000)])
def test_latent_precision(rows, heads, keys):
    print("latent rms", rows, heads, keys, flush=True)
    g = torch.Generator(device=DEV).manual_seed(keys)
    pool, q = latent.rand_pool(g, 10000), latent.rand_q(g, rows, heads)
    ids = torch.randint(0, 10000, (rows, keys), device=DEV, generator=g, dtype=I32)
    out = LT.attend(q, pool, ids)
    some = list(range(0, rows, max(1, rows // 20)))
    ref = torch.stack([latent.reference(q[r], pool, ids[r], 192 ** -0.5)[0] for r in some])
    got, rounded = errors(out[some], ref)
    print(got / rounded, flush=True)
    # (a work-group of up to 32 heads: two bf16 numbers a probability; the 128 heads of 300 rows go 64 a work-group, one number)
    assert got <= (1.1 if heads <= 32 else 1.5) * rounded, got / rounded


@gpu
def test_kv8_and_expanded_precision():
    print("kv8, expanded rms", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    (kp, ks), (vp, vs) = kv8.rand_pool(g, 100, 2), kv8.rand_pool(g, 100, 2)
    q = torch.randn((20, 16, 128), device=DEV, generator=g).to(BF16)
    ids = torch.randint(0, 6400, (20, 1000), device=DEV, generator=g, dtype=I32)
    out = K8.attend(q, kp, vp, ks, vs, torch.arange(100, device=DEV, dtype=I32), ids=ids)
    at = ids.long()
    ref = torch.stack([torch.cat([kv8.reference(q[r, 8 * h:8 * h + 8], [kp, vp, ks, vs], at[r] // 64, at[r] % 64, h, 128 ** -0.5)[0] for h in range(2)])
                       for r in range(20)])
    got, rounded = errors(out, ref)
    print(got / rounded, flush=True)
    assert got <= 1.1 * rounded
    r = lambda *s: torch.randn(s, device=DEV, generator=g).to(BF16)
    q, kv, rope = r(300, 4, 192), r(1500, 4, 256), r(1500, 64)
    cu = lambda n: torch.tensor([0, n], device=DEV, dtype=I32)
    out = LT.attend_expanded(q, kv, rope, cu(300), cu(1500), 300, causal=False)
    k = torch.cat([kv[..., :128], rope[:, None].expand(-1, 4, -1)], 2).double()
    s = 192 ** -0.5 * torch.matmul(q.double().transpose(0, 1), k.permute(1, 2, 0).contiguous())
    ref = torch.matmul(torch.softmax(s, -1), kv[..., 128:].double().transpose(0, 1).contiguous()).transpose(0, 1)
    got, rounded = errors(out, ref)
    print(got / rounded, flush=True)
    assert got <= 1.5 * rounded
