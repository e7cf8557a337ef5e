"""The operators over K/V pages of 16-bit numbers as they are used: step after step of
a request's life, captured into graphs, on other streams and threads, with long
contexts, far strides and the ends of the number range.  Bounds as in test_gpu_paged."""
import math
import threading

import pytest
import torch

from conftest import pkg
from test_gpu_paged import BF16, DEV, F16, I32, PG, check, chains, gen, make, offsets, random_tree, rows_of, run_and_check, seen_and_distance

gpu = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def rotated(x, rot, at, interleaved=False):
    """In float64, rounded once more by the caller's bound."""
    cos, sin = rot[at].double().chunk(2, 1)
    half = cos.shape[1]
    i = torch.arange(half, device=DEV)
    re, im = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.double().clone()
    a, b = x.double()[..., re], x.double()[..., im]
    y[..., re], y[..., im] = a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]
    return y


# ------------------------------------------------------------------ together
@gpu
@pytest.mark.parametrize("kv_heads,group,dtype", [(2, 4, BF16), (1, 6, F16)])
def test_a_request_from_prompt_to_accepted_drafts(kv_heads, group, dtype):
    """Prompts appended and attended, a tree of drafts behind them, the accepted path kept, the next token attended: each
    against a plain cache in which the rows lie in order."""
    print("life", kv_heads, group, dtype, flush=True)
    g, heads = gen(21), kv_heads * group
    prompts, pages = [70, 5, 200], 40
    pools = [torch.full((pages, 64, kv_heads, 128), math.nan, device=DEV, dtype=dtype) for _ in range(2)]
    table = torch.randperm(pages, device=DEV, generator=g)[:30].view(3, 10).to(I32)
    rot = PG.rotations(1000, device=DEV)
    kept = [[torch.zeros((0, kv_heads, 128), device=DEV, dtype=dtype) for _ in range(2)] for _ in prompts]  # the plain cache

    def new(n):
        return [torch.randn((n, h, 128), device=DEV, generator=g).to(dtype) for h in (heads, kv_heads, kv_heads)]

    def stored(counts, starts, at, q, k, v):
        """Appends, and checks the pages' new rows; the rotated queries and rows, by request."""
        out = PG.append(q, k, v, *pools, table, i32(starts), offsets(counts), rot, i32(at))
        u, t, per = torch.finfo(dtype).eps / 2, 0, []
        want_q, want_k = rotated(q, rot, torch.tensor(at, device=DEV)), rotated(k, rot, torch.tensor(at, device=DEV))
        assert bool(((out.double() - want_q).abs() <= u * want_q.abs() + 2.0 ** -20).all())
        for r, n in enumerate(counts):
            rows = [rows_of(pool, table[r], starts[r] + n)[starts[r]:] for pool in pools]
            assert bool(((rows[0].double() - want_k[t:t + n]).abs() <= u * want_k[t:t + n].abs() + 2.0 ** -20).all())
            assert torch.equal(rows[1], v[t:t + n])
            per.append((out[t:t + n], *rows))
            t += n
        return out, per

    # prompts
    q, k, v = new(sum(prompts))
    out, per = stored(prompts, [0, 0, 0], [i for n in prompts for i in range(n)], q, k, v)
    got, lse = PG.attend(out, *pools, table, i32(prompts), offsets(prompts), max(prompts), softcap=20.0, return_lse=True)
    t = 0
    for r, n in enumerate(prompts):
        kept[r] = [per[r][1], per[r][2]]
        check(got[t:t + n], lse[t:t + n], per[r][0], *kept[r], *seen_and_distance(n, n), cap=20.0)
        t += n
    for step in range(3):
        # drafts
        lens = [x[0].shape[0] for x in kept]
        counts = [9, 1, 17]
        trees = [random_tree(n, 10 * step + n) for n in counts]
        depths = [[len(c) - 1 for c in chains(tree)] for tree in trees]
        q, k, v = new(sum(counts))
        out, per = stored(counts, lens, [lens[r] + d for r, x in enumerate(depths) for d in x], q, k, v)
        got, lse = PG.attend_tree(out, *pools, table, i32([a + b for a, b in zip(lens, counts)]), i32(sum(trees, [])), offsets(counts), 17,
                                  softcap=20.0, window=100, return_lse=True)
        t, accepted = 0, []
        for r, n in enumerate(counts):
            rows = [torch.cat([kept[r][i], per[r][i + 1]]) for i in range(2)]
            check(got[t:t + n], lse[t:t + n], per[r][0], *rows, *seen_and_distance(n, lens[r] + n, 100, parents=trees[r]), cap=20.0)
            accepted.append(chains(trees[r])[n - 1][::-1])
            kept[r] = [torch.cat([kept[r][i], per[r][i + 1][accepted[r]]]) for i in range(2)]
            t += n
        PG.keep(*pools, table, i32(lens), i32(sum(accepted, [])), offsets([len(a) for a in accepted]))
        # one token each
        lens = [x[0].shape[0] for x in kept]
        for r, n in enumerate(lens):
            assert all(torch.equal(rows_of(pool, table[r], n), x) for pool, x in zip(pools, kept[r])), (step, r)
        q, k, v = new(3)
        out, per = stored([1, 1, 1], lens, lens, q, k, v)
        kept = [[torch.cat([x, y]) for x, y in zip(kept[r], per[r][1:])] for r in range(3)]
        got, lse = PG.attend(out, *pools, table, i32([n + 1 for n in lens]), softcap=20.0, return_lse=True)
        for r, n in enumerate(lens):
            check(got[r:r + 1], lse[r:r + 1], out[r:r + 1], *kept[r], *seen_and_distance(1, n + 1), cap=20.0)


# -------------------------------------------------------------- graphs and streams
@gpu
@pytest.mark.parametrize("drafts,group", [(3, 4), (20, 8)])
def test_captured_steps_with_lengths_that_change(drafts, group):
    """append -> attend_tree -> keep captured, replayed with other lengths, tables and tokens between eager calls."""
    print("graph", drafts, group, flush=True)
    g, requests, kv_heads = gen(31), 5, 2
    heads, tokens = kv_heads * group, requests * drafts
    shape = (200, 64, kv_heads, 128)
    pools = [torch.randn(shape, device=DEV, generator=g).to(BF16) for _ in range(2)]
    table = torch.zeros((requests, 36), device=DEV, dtype=I32)
    starts, lens, parents = (torch.zeros(n, device=DEV, dtype=I32) for n in (requests, requests, tokens))
    positions, ids = torch.zeros(tokens, device=DEV, dtype=I32), torch.zeros(2 * requests, device=DEV, dtype=I32)
    q = torch.zeros((tokens, heads, 128), device=DEV, dtype=BF16)
    k, v = (torch.zeros((tokens, kv_heads, 128), device=DEV, dtype=BF16) for _ in range(2))
    rot, cu, cu_ids = PG.rotations(3000, device=DEV), offsets([drafts] * requests), offsets([2] * requests)

    def step(pools):
        out = PG.append(q, k, v, *pools, table, starts, cu, rot, positions)
        got = PG.attend_tree(out, *pools, table, lens, parents, cu, drafts, softcap=10.0, return_lse=True)
        PG.keep(*pools, table, starts, ids, cu_ids)
        return got

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(pools)
    for replay in range(4):
        older = torch.randint(0, 2200 if replay % 2 else 150, (requests,), device=DEV, generator=g, dtype=I32)
        table.copy_(torch.randperm(200, device=DEV, generator=g)[:180].view(requests, 36))
        starts.copy_(older)
        lens.copy_(older + drafts)
        trees = [random_tree(drafts, 100 * replay + r) for r in range(requests)]
        parents.copy_(i32(sum(trees, [])))
        depth = [len(c) - 1 for tree in trees for c in chains(tree)]
        positions.copy_(older.repeat_interleave(drafts) + i32(depth))
        ids.copy_(i32([x for r in range(requests) for x in (0, 1 + (r + replay) % (drafts - 1))]))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV, generator=g))
        eager = [x.clone() for x in pools]
        want, want_lse = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse), replay
        assert all(torch.equal(a, b) for a, b in zip(pools, eager)), replay
        PG.attend(q[:requests], *pools, table, lens)  # (eager work of its own between the replays)


@gpu
def test_two_graphs_replayed_side_by_side():
    """Their workspaces are their own."""
    g = gen(32)
    graphs, outs, wants, inputs = [], [], [], []
    for i in range(2):
        (kp, vp), table = make(g, [3000 + 500 * i, 100], 1, BF16)
        q = torch.randn((2, 8, 128), device=DEV, generator=g).to(BF16)
        lens = i32([3000 + 500 * i, 100])
        inputs.append((q, kp, vp, table, lens))  # (a graph reads them where they were: they stay for its replays)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(PG.attend(q, kp, vp, table, lens))
        graphs.append(graph)
        wants.append(PG.attend(q, kp, vp, table, lens))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))


@gpu
def test_other_streams_and_threads():
    g = gen(33)
    (kp, vp), table = make(g, [2500, 700, 64], 2, F16)
    lens = i32([2500, 700, 64])
    q = torch.randn((90, 8, 128), device=DEV, generator=g).to(F16)
    cu = offsets([30, 30, 30])
    want = PG.attend(q, kp, vp, table, lens, cu, 30), PG.attend(q[:3], kp, vp, table, lens)
    torch.cuda.synchronize()
    bad = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = PG.attend(q, kp, vp, table, lens, cu, 30), PG.attend(q[:3], kp, vp, table, lens)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ----------------------------------------------------------------- long contexts
@gpu
def test_more_than_64_tiles_of_a_wave():
    """300 requests over one table of 300 pages, the last of the keys of each its own length."""
    g = gen(41)
    (kp, vp), table = make(g, [19200], 1, BF16, fill=0.0)
    lens = torch.randint(18000, 19201, (300,), generator=g, device=DEV).to(I32)
    q = torch.randn((300, 2, 128), device=DEV, generator=g).to(BF16)
    out, lse = PG.attend(q, kp, vp, table.expand(300, -1)[:, :300], lens, return_lse=True)
    k, v = rows_of(kp, table[0], 19200), rows_of(vp, table[0], 19200)
    for r in range(0, 300, 37):
        n = int(lens[r])
        check(out[r:r + 1], lse[r:r + 1], q[r:r + 1], k[:n], v[:n], *seen_and_distance(1, n))


@gpu
@pytest.mark.parametrize("more", [dict(), dict(slopes=True), dict(window=5000, prefix=[700])])
def test_more_than_64_tiles_of_a_block(more):
    print("long", more, flush=True)
    run_and_check(gen(42), [1000], [9000], 8, 8, BF16, **more)


@gpu
def test_parts_of_many_queries():
    """A few queries' blocks over long contexts: every request's keys in many parts, one request without any."""
    for tree in (None, [random_tree(40, 1), random_tree(3, 2), random_tree(64, 3)]):
        run_and_check(gen(43), [40, 3, 64], [20000, 3, 6000], 1, 4, F16, tree=tree)
    run_and_check(gen(44), [40, 3], [12000, 9000], 1, 4, BF16, window=300, prefix=[5000, 10])  # (parts that see nothing)


@gpu
def test_offsets_past_32_bits():
    """Pages 2^31 numbers apart, tokens of a page 2^25 - 8 apart; positions of a table of 2^24 entries."""
    n, kinds = 100, []
    g = gen(45)
    (kp, vp), table = make(g, [n], 1, BF16)
    q = torch.randn((40, 4, 128), device=DEV, generator=g).to(BF16)
    lens, cu = i32([n]), offsets([40])
    want = PG.attend(q, kp, vp, table, lens, cu), PG.attend(q[:1], kp, vp, table, lens)
    order = table[0, :2].long()
    for page, token in ((1 << 31, 128), (128, (1 << 25) - 8)):
        far = []
        for pool in (kp, vp):
            storage = torch.empty(page + 63 * token + 128, device=DEV, dtype=BF16)
            x = storage.as_strided((2, 64, 1, 128), (page, token, 128, 1))
            x.copy_(pool[order])
            far.append(x)
        t = i32([[0, 1]])
        for a, b in zip(want, (PG.attend(q, *far, t, lens, cu), PG.attend(q[:1], *far, t, lens))):
            assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7  # (the table's length decides the parts)
        PG.keep(*far, t, i32([0]), i32([0, 99]), i32([0, 2]))
        assert torch.equal(far[0][0, 1], kp[order[1], 35]) and torch.equal(far[1][0, 1], vp[order[1], 35])
        new = torch.randn((1, 1, 128), device=DEV, generator=g).to(BF16)
        PG.append(None, new, new, *far, t, i32([101]), i32([0, 1]), PG.rotations(200, device=DEV))
        assert torch.equal(far[1][1, 37], new[0])
        del far, x, storage
        torch.cuda.empty_cache()
    # a context of 2^30 positions, whose pages are one and the same, seen through a window and a prefix
    wide = torch.zeros((1, 1 << 24), device=DEV, dtype=I32)
    wide[0, 0], wide[0, -1] = order[0], order[0]
    wide[0, 1:-1] = -1
    out, lse = PG.attend(q[:1], kp, vp, wide, i32([1 << 30]), window=64, prefix=i32([64]), return_lse=True)
    k, v = (torch.cat([pool[order[0]]] * 2) for pool in (kp, vp))
    check(out, lse, q[:1], k, v, torch.ones((1, 128), dtype=torch.bool, device=DEV), torch.zeros((1, 128), device=DEV))


# --------------------------------------------------------------- ends of the range
@gpu
@pytest.mark.parametrize("nq,group", [(1, 4), (100, 2)])
@pytest.mark.parametrize("dtype,big", [(BF16, 2.0 ** 90), (F16, 60000.0)])
def test_large_and_small_values(nq, group, dtype, big):
    """Values to the top of the types' range, and a key that outweighs thousands of others by 2^20."""
    print("range", nq, group, dtype, big, flush=True)
    g, n = gen(51), 3000
    (kp, vp), table = make(g, [n], 1, dtype)
    q = torch.randn((nq, group, 128), device=DEV, generator=g).to(dtype)
    page, row = table[0, 10].long(), 3
    k = kp[page, row, 0]
    k.copy_(q[0, 0].float() * 14.0 / q[0, 0].float().pow(2).sum() * 128 ** 0.5)  # (scores 14 with the first column)
    vp[table[0, :46].long()] *= big / 8
    vp[torch.isnan(vp)] = 0
    vp.clamp_(-big, big)
    out, lse = PG.attend(q, kp, vp, table, i32([n]), offsets([nq]), return_lse=True)
    check(out, lse, q, rows_of(kp, table[0], n), rows_of(vp, table[0], n), *seen_and_distance(nq, n))


@gpu
@pytest.mark.parametrize("cap,scale", [(1e-30, 0.1), (1e-3, 0.1), (30.0, 1e-6), (30.0, 30.0), (1e30, 0.1), (1e5, 1e-25), (0.5, 0.088)])
@pytest.mark.parametrize("slopes", [False, True])
def test_caps_far_from_the_scale(cap, scale, slopes):
    """(1e30 of 0.1: scores as without a cap.)"""
    print("caps", cap, scale, slopes, flush=True)
    run_and_check(gen(52), [1, 60], [300, 100], 1, 4, BF16, cap=cap, scale=scale, slopes=slopes)


@gpu
def test_slopes_of_all_sizes():
    """Distances that hide all but the nearest keys, none, and ones that favour far keys."""
    g, n, nq = gen(53), 2000, 70
    (kp, vp), table = make(g, [n], 1, BF16)
    q = torch.randn((nq, 6, 128), device=DEV, generator=g).to(BF16)
    slopes = torch.tensor([100.0, 1.0, 0.0, 1e-6, -0.01, -3.0], device=DEV)
    for first in (0, nq - 1):
        out, lse = PG.attend(q[first:], kp, vp, table, i32([n]), offsets([nq - first]), slopes=slopes, return_lse=True)
        seen, away = seen_and_distance(nq - first, n)
        check(out, lse, q[first:], rows_of(kp, table[0], n), rows_of(vp, table[0], n), seen, away, slopes=slopes)


@gpu
def test_the_same_bits_again():
    """No sum depends on the order in which work-groups end."""
    g = gen(54)
    (kp, vp), table = make(g, [9000, 4000, 300], 2, BF16)
    q = torch.randn((93, 8, 128), device=DEV, generator=g).to(BF16)
    lens, cu = i32([9000, 4000, 300]), offsets([31, 31, 31])
    for call in (lambda: PG.attend(q, kp, vp, table, lens, cu, 31, return_lse=True), lambda: PG.attend(q[:3], kp, vp, table, lens, return_lse=True)):
        want = call()
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(call(), want))


@gpu
@pytest.mark.parametrize("nq,group", [(1, 4), (90, 2)])
def test_subnormal_numbers(nq, group):
    """fp16 keys and values below its normal numbers: the products keep them (an output is then off by half of
    the smallest number, 2^-25, beside the bound)."""
    g, n = gen(55), 300
    (kp, vp), table = make(g, [n], 1, F16)
    for pool, by in ((kp, 2.0 ** -18), (vp, 2.0 ** -20)):
        pool.copy_(pool.float() * by)
    q = torch.randn((nq, group, 128), device=DEV, generator=g).to(F16)
    out, lse = PG.attend(q, kp, vp, table, i32([n]), offsets([nq]), softmax_scale=2.0 ** 14, return_lse=True)
    k, v = rows_of(kp, table[0], n).double(), rows_of(vp, table[0], n).double()
    seen, _ = seen_and_distance(nq, n)
    s = 2.0 ** 14 * torch.einsum("qhd,kd->qhk", q.double(), k[:, 0]).masked_fill(~seen[:, None], -math.inf)
    d = (128 + 8) * 2.0 ** -24 * 2.0 ** 14 * torch.einsum("qhd,kd->qhk", q.double().abs(), k[:, 0].abs()).amax(-1)
    want_lse = torch.logsumexp(s, -1)
    p = torch.exp(s - want_lse[..., None])
    want, mag, u = p @ v[:, 0], p @ v[:, 0].abs(), 2.0 ** -11
    assert bool(((out.double() - want).abs() <= u * (want.abs() + mag) * (1 + u) + 2 * d[..., None] * mag + 2.0 ** -25 + n * 2.0 ** -31 * v.abs().amax()).all())
    assert bool(((lse.double() - want_lse).abs() <= d + 2.0 ** -21 * (1 + want_lse.abs() + s.masked_fill(~seen[:, None], 0).abs().amax(-1))).all())
