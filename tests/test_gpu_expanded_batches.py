"""Attention over expanded keys and values where the batch's sequences are far from
alike: lengths not given on the host, many short sequences, long ones among short
ones, padded buffers.  Against float64 with the bounds of the operator's own tests,
and against the same sequences in calls that know their lengths (a block of queries
does the same sums wherever it lies in the launch, so those are equal)."""
import random

import pytest
import torch

import test_gpu_expanded as expanded
from conftest import pkg

LT = pkg("latent")
DEV = "cuda:0"
gpu = pytest.mark.gpu


def lengths(kind, n):
    rng = random.Random(n)
    if kind == "short":
        return [rng.choice([0, 1, 2, 7, 64, 100]) for _ in range(n)]
    if kind == "one long":
        return [rng.choice([0, 1, 90]) for _ in range(n // 2)] + [5000] + [rng.choice([0, 1, 256, 257]) for _ in range(n // 2)]
    return [rng.choice([0, 1, 255, 256, 257, 511, 513, 900]) for _ in range(n)]


@gpu
@pytest.mark.parametrize("n", [2, 9, 63, 64, 65, 130, 700])
@pytest.mark.parametrize("kind", ["short", "one long", "mixed"])
@pytest.mark.parametrize("causal", [True, False])
def test_batches_without_max_q(n, kind, causal):
    print("expanded batch", n, kind, causal, flush=True)
    nq = lengths(kind, n)
    nk = [max(0, m + (17, 0, -3, 400)[i % 4]) for i, m in enumerate(nq)]
    q, kv, rope, cu_q, cu_k = expanded.inputs(n, nq, nk, 2, behind=300)
    out = torch.full((q.shape[0], 2, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    _, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, causal=causal, out=out, return_lse=True)
    assert bool((out[sum(nq):] == 7).all())
    known, known_lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max(nq), causal=causal, return_lse=True)
    if n >= 63:  # (too few keys a sequence for parts, either way)
        assert torch.equal(out[:sum(nq)], known[:sum(nq)]) and torch.equal(lse[:sum(nq)], known_lse[:sum(nq)])
    few = sorted(random.Random(1).sample(range(len(nq)), min(len(nq), 12)) + [nq.index(max(nq))])
    for b in few:
        i, j = int(cu_q[b]), int(cu_k[b])
        for o, l in ((out, lse), (known, known_lse)):
            expanded.check(o[i:i + nq[b]], l[i:i + nq[b]], q[i:i + nq[b]], kv[j:j + nk[b]], rope[j:j + nk[b]], [nq[b]], [nk[b]], causal)


@gpu
def test_sequences_that_begin_behind_the_first_row():
    """Rows before the first sequence, and a batch that ends before the buffer does."""
    print("expanded begin", flush=True)
    for n, first in ((70, 1000), (3, 300), (1, 256)):
        nq = [1, 300, 40] * 30
        nq = nq[:n]
        q, kv, rope, cu, _ = expanded.inputs(n, nq, nq, 2, behind=4000)
        out = torch.full((q.shape[0], 2, 128), 7.0, device=DEV, dtype=torch.bfloat16)
        want, want_lse = LT.attend_expanded(q[first:], kv[first:], rope[first:], cu, return_lse=True)
        _, lse = LT.attend_expanded(q, kv, rope, cu + first, out=out, return_lse=True)
        end = first + sum(nq)
        assert bool((out[:first] == 7).all()) and bool((out[end:] == 7).all())
        expanded.check(out[first:end], lse[first:end], q[first:], kv[first:], rope[first:], nq, nq)
        expanded.check(want[:sum(nq)], want_lse[:sum(nq)], q[first:], kv[first:], rope[first:], nq, nq)


@gpu
def test_more_blocks_than_a_launch_holds():
    """2048 sequences whose lengths only the device knows, 512 heads: a block of the
    longest possible for each would be more work-groups than a launch can have."""
    print("expanded launch", flush=True)
    heads, nq = 512, [(1, 0, 2, 1)[i % 4] for i in range(2047)] + [60]
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(s, device=DEV, generator=g, dtype=torch.bfloat16)
    q, kv, rope = r(sum(nq) + 600, heads, 192), r(sum(nq), heads, 256), r(sum(nq), 64)
    cu = torch.tensor([0] + nq, device=DEV).cumsum(0).to(torch.int32)
    assert len(nq) * -(-q.shape[0] // 256) * heads >= (1 << 32) // 512
    out, lse = LT.attend_expanded(q, kv, rope, cu, return_lse=True)
    n = sum(nq)
    known, known_lse = LT.attend_expanded(q, kv, rope, cu, max_q=60, return_lse=True)
    assert torch.equal(out[:n], known[:n]) and torch.equal(lse[:n], known_lse[:n])
    for b in (0, 1, 2, 1000, 2046, 2047):
        i = int(cu[b])
        pick = lambda t: t[i:i + nq[b], 5::100]
        expanded.check(pick(out), pick(lse), pick(q), pick(kv), rope[i:i + nq[b]], [nq[b]], [nq[b]])


@gpu
@pytest.mark.parametrize("max_q", [1, 100, 256, 257, 1500])
@pytest.mark.parametrize("heads,nq", [(1, [900]), (1, [90, 0, 3000, 300]), (40, [700, 20, 1600]), (2, [3, 40, 1] * 30 + [4000] + [5, 257] * 20)])
@pytest.mark.parametrize("causal", [True, False])
def test_only_the_first_max_q_queries(heads, nq, max_q, causal):
    """Each sequence's first max_q queries, at their places before the end of its
    keys; every other row of the output is left alone."""
    print("expanded max_q", heads, len(nq), max_q, causal, flush=True)
    nk = [n + (0, 30, -1)[i % 3] for i, n in enumerate(nq)]
    nk = [max(0, m) for m in nk]
    q, kv, rope, cu_q, cu_k = expanded.inputs(max_q, nq, nk, heads)
    out = torch.full((sum(nq), heads, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    _, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max_q, causal=causal, out=out, return_lse=True)
    whole, whole_lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, causal=causal, return_lse=True)
    some = torch.cat([torch.arange(n, device=DEV) < max_q for n in nq])
    assert bool((out[~some] == 7).all())
    whole[some], whole_lse[some] = out[some], lse[some]
    for h in range(0, heads, 9):
        expanded.check(whole[:, h:h + 1], whole_lse[:, h:h + 1], q[:, h:h + 1], kv[:, h:h + 1], rope, nq, nk, causal)


@gpu
@pytest.mark.parametrize("nq,nk,max_q,heads,behind", [
    ([200], [20000], 200, 2, 100000), ([1], [3000], 1, 16, 100000), ([3, 0, 70, 1], [5000, 40, 900, 0], 70, 2, 100000),
    ([3, 0, 90, 1], [5000, 40, 900, 1], 70, 2, 100000), ([400, 300], [9000, 8000], 400, 1, 100000),
    ([1] * 40 + [900] + [2] * 20, [3000] * 61, 900, 1, 100000), ([1] * 40 + [900] + [2] * 20, [3000] * 61, 900, 1, 0)])
def test_parts_of_a_padded_buffer(nq, nk, max_q, heads, behind):
    """Few queries in a buffer for many, their keys in several parts (but for the last
    batch with its padding, whose blocks could be as many as the CUs): the sums take
    the room of the sequences or of the tokens, and rows outside the sequences stay."""
    print("expanded padded", nq[:4], max_q, behind, flush=True)
    L = pkg("_lib")
    first = 9
    need = L.lib().v1_latent_expanded_workspace(sum(nq) + behind + first, sum(nk), len(nq), heads, max_q)
    assert need <= (1 << 16) * 130 * 4 and (need > 0) == (max_q < 900 or behind == 0), need
    q, kv, rope, cu_q, cu_k = expanded.inputs(7, nq, nk, heads)
    wide = torch.full((sum(nq) + behind + first, heads, 192), float("nan"), device=DEV, dtype=torch.bfloat16)
    wide[first:first + sum(nq)] = q
    out = torch.full((wide.shape[0], heads, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    _, lse = LT.attend_expanded(wide, kv, rope, cu_q + first, cu_k, max_q, out=out, return_lse=True)
    some = torch.zeros(wide.shape[0], device=DEV, dtype=torch.bool)
    some[first:first + sum(nq)] = torch.cat([torch.arange(n, device=DEV) < max_q for n in nq])
    assert bool((out[~some] == 7).all())
    whole, whole_lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, return_lse=True)
    mine = some[first:first + sum(nq)]
    whole[mine], whole_lse[mine] = out[some], lse[some]
    expanded.check(whole, whole_lse, q, kv, rope, nq, nk)


@gpu
@pytest.mark.parametrize("batch,tokens,keys,max_q,heads", [(70, 3000, 3000, None, 2), (3, 20000, 9000, 40, 2), (61, 1000, 60000, 900, 1)])
def test_graphs_whose_lengths_change(batch, tokens, keys, max_q, heads):
    """Captured once (slots; a padded buffer in parts; slots in parts) and replayed with
    other sequences, lengths of 0 and rows behind the last one among them."""
    print("expanded graph", batch, max_q, flush=True)
    rng = random.Random(batch)
    q, kv, rope, _, _ = expanded.inputs(batch, [tokens], [keys], heads)
    cu_q, cu_k = (torch.zeros(batch + 1, device=DEV, dtype=torch.int32) for _ in range(2))
    out = torch.zeros((tokens, heads, 128), device=DEV, dtype=torch.bfloat16)

    def refill():
        most = min(max_q or tokens, tokens // batch)
        nq = [rng.choice([0, 1, rng.randint(0, most), most]) for _ in range(batch)]
        if batch > 3:
            nq[rng.randrange(batch)] = (max_q or 1500) // 2
        nk = [rng.randint(0, keys // batch) for _ in nq]
        for cu, n in ((cu_q, nq), (cu_k, nk)):
            cu.copy_(torch.tensor([0] + n).cumsum(0))
        out.fill_(7.0)
        return nq, nk

    refill()
    LT.attend_expanded(q, kv, rope, cu_q, cu_k, max_q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max_q, out=out, return_lse=True)
    for _ in range(4):
        nq, nk = refill()
        n = sum(nq)
        assert n <= tokens
        want, want_lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max_q, return_lse=True)
        torch.randn(1 << 20, device=DEV).sort()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:n], want[:n]) and torch.equal(lse[:n], want_lse[:n]) and bool((out[n:] == 7).all())
        b = nq.index(max(nq))
        i, j = int(cu_q[b]), int(cu_k[b])
        expanded.check(out[i:i + nq[b]], lse[i:i + nq[b]], q[i:i + nq[b]], kv[j:j + nk[b]], rope[j:j + nk[b]], [nq[b]], [nk[b]])


def test_room_for_parts():
    """Never more than 256 rows of sums for each work-group of one round."""
    L = pkg("_lib")
    if not L.LIB_PATH.exists():
        pkg("build").build()
    room = L.lib().v1_latent_expanded_workspace
    for tokens in (1, 200, 8192, 100000, 1 << 20):
        for batch in (1, 3, 60):
            for max_q in (1, 200, 300, 5000, tokens):
                for heads in (1, 16, 100):
                    for keys in (100, 65536, 1 << 24):
                        assert room(tokens, keys, batch, heads, min(max_q, tokens)) <= (1 << 16) * 130 * 4, (tokens, keys, batch, heads, max_q)
    assert room(8192, 65536, 1, 16, 200) == room(200, 65536, 1, 16, 200) > 0
    assert room(16384, 1 << 20, 1, 1, 1) == room(1, 1 << 20, 1, 1, 1) > 0


def library_call(**change):
    L = pkg("_lib")
    if not L.LIB_PATH.exists():
        pkg("build").build()
    base = dict(q=256, qr=384, qh=192, kv=256, kr=512, kh=256, rope=256, rr=64, cu_q=256, cu_k=256, out=256, o_row=256, o_head=128,
                lse=0, ws=0, wsb=0, tokens=4096, keys=4096, batch=1, heads=16, max_q=4096, causal=1, scale=0.1)
    return L.lib().v1_latent_expanded(L.PACKED["v1_latent_expanded"].pack(*{**base, **change}.values()), None), L


def test_too_many_sequences_for_a_launch():
    for change in (dict(batch=1 << 16, heads=128, max_q=1), dict(batch=1 << 17, heads=64), dict(batch=(1 << 31) - 1, heads=1),
                   dict(batch=(1 << 31) - 1, heads=65535, tokens=1 << 30, max_q=1 << 30)):
        rc, L = library_call(**change)
        assert rc == L.V1_ERR_INVALID and b"launch" in L.lib().v1_last_error(), change
