"""K / V pages of 16-bit numbers: tokens appended with their keys rotated, and rows moved.

Bound of a rotated number x cos - y sin, u = eps / 2 of its type: fp32 products and sum
are off by 3 2^-24 (|x cos| + |y sin|) at most, then one rounding:
  |got - ref| <= u |ref| + 2^-22 (|x cos| + |y sin|) (1 + u)  (+ half of the smallest number)."""
import math

import pytest
import torch

from conftest import pkg

PG = pkg("paged")
DEV = "cuda:0"
gpu = pytest.mark.gpu
BF16, F16, I32 = torch.bfloat16, torch.float16, torch.int32


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def offsets(counts):
    return i32([0, *torch.tensor(counts).cumsum(0).tolist()])


def turned(x, cos, sin, interleaved):
    """x [tokens, heads, 128] -> value and bound's magnitude, float64."""
    half = cos.shape[1]
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    i = torch.arange(half, device=DEV)
    re, im = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., re], y[..., im] = x[..., re] * cos - x[..., im] * sin, x[..., im] * cos + x[..., re] * sin
    mag[..., re] = (x[..., re] * cos).abs() + (x[..., im] * sin).abs()
    mag[..., im] = (x[..., im] * cos).abs() + (x[..., re] * sin).abs()
    return y, mag


def close(got, ref, mag, dtype):
    u = torch.finfo(dtype).eps / 2
    bound = u * ref.abs() + 2.0 ** -22 * mag * (1 + u) + torch.finfo(dtype).smallest_normal * u
    return bool(((got.double() - ref).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("starts,new", [([0], [1]), ([63, 5, 64], [2, 0, 70]), ([100, 0, 200, 7], [1, 1, 1, 1]), ([1, 130], [300, 65])])
@pytest.mark.parametrize("heads,kv_heads,rotated,interleaved,dtype,major", [
    (4, 1, 128, False, BF16, "token"), (32, 8, 128, True, F16, "head"), (3, 3, 64, False, F16, "token"), (5, 1, 16, True, BF16, "head"),
    (0, 2, 96, False, BF16, "token"), (8, 2, 112, False, BF16, "token"), (7, 7, 128, False, BF16, "head")])
@pytest.mark.parametrize("own_positions", [False, True])
def test_append(starts, new, heads, kv_heads, rotated, interleaved, dtype, major, own_positions):
    print("append", starts, new, heads, kv_heads, rotated, interleaved, dtype, major, own_positions, flush=True)
    g = torch.Generator(device=DEV).manual_seed(sum(starts) + heads)
    tokens, pages = sum(new), 60
    shape = (pages, 64, kv_heads, 128) if major == "token" else (pages, kv_heads, 64, 128)
    pools = [torch.randn(shape, device=DEV, generator=g).to(dtype) for _ in range(2)]
    pools = [x if major == "token" else x.transpose(1, 2) for x in pools]
    before = [x.clone() for x in pools]
    table = torch.randperm(pages, device=DEV, generator=g)[:10 * len(starts)].view(-1, 10).to(I32)
    k, v = (torch.randn((tokens, kv_heads, 128), device=DEV, generator=g).to(dtype) for _ in range(2))
    q = torch.randn((tokens, heads, 128), device=DEV, generator=g).to(dtype) if heads else None
    rot = PG.rotations(700, rotated, device=DEV)
    position = [s + i for s, n in zip(starts, new) for i in range(n)]
    angle = [(p * 7 + 3) % 700 for p in position] if own_positions else position
    got = PG.append(q, k, v, *pools, table, i32(starts), offsets(new), rot, i32(angle) if own_positions else None, interleaved)
    cos, sin = rot[torch.tensor(angle, device=DEV)].chunk(2, 1)
    if heads:
        ref, mag = turned(q, cos, sin, interleaved)
        assert close(got, ref, mag, dtype) and torch.equal(got[..., rotated:], q[..., rotated:])
    else:
        assert got is None
    of = torch.tensor([r for r, n in enumerate(new) for _ in range(n)], device=DEV)
    at = torch.tensor(position, device=DEV)
    page, row = table[of, at // 64].long(), at % 64
    ref, mag = turned(k, cos, sin, interleaved)
    assert close(pools[0][page, row], ref, mag, dtype) and torch.equal(pools[0][page, row][..., rotated:], k[..., rotated:])
    assert torch.equal(pools[1][page, row], v)
    for pool, was in zip(pools, before):
        was[page, row] = pool[page, row]
        assert torch.equal(pool, was)


@gpu
def test_append_skips():
    """Tokens outside the requests, without an angle, with a negative start, past the table, in pages outside the pool."""
    g = torch.Generator(device=DEV).manual_seed(2)
    new, lead = [3, 2, 4, 70, 2], 2
    tokens = lead + sum(new) + 3
    k, v = (torch.randn((tokens, 2, 128), device=DEV, generator=g).to(BF16) for _ in range(2))
    q = torch.randn((tokens, 4, 128), device=DEV, generator=g).to(BF16)
    pools = [torch.randn((20, 64, 2, 128), device=DEV, generator=g).to(BF16) for _ in range(2)]
    before = [x.clone() for x in pools]
    table = i32([[0, 1], [2, 3], [-1, 20], [4, 5], [6, 7]])
    starts = i32([10, -1, 62, 100, 299])
    cu = offsets(new) + lead
    out = torch.full_like(q, 5.0)
    rot = PG.rotations(300, device=DEV)
    PG.append(q, k, v, *pools, table, starts, cu, rot, out=out)
    # request 0 is stored; 1 begins below zero; 2's pages are not there; of 3 positions 100 .. 127; of 4 position 299 is past the table
    written = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    written[2:5] = True                  # request 0
    written[6] = True                    # request 1's second token has angle 0
    written[7:11] = True                 # request 2: rotated, not stored
    written[11:81] = True                # request 3
    written[81] = True                   # request 4: angle 299; 300 is not in the table
    assert bool((out[~written] == 5).all()) and not bool((out[written] == 5).all(-1).any())
    want = before[1].clone()
    want[0, 10:13] = v[2:5]
    want[5, 36:64] = v[11:39]
    assert torch.equal(pools[1], want)
    same = torch.ones_like(want, dtype=torch.bool)
    same[0, 10:13], same[5, 36:64] = False, False
    assert torch.equal(pools[0][same], before[0][same]) and not torch.equal(pools[0], before[0])


@gpu
def test_append_in_place_and_strided():
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.randn((90, 8 + 4, 128), device=DEV, generator=g).to(BF16)   # a projection's output: q, k, v side by side
    pools = [torch.zeros((9, 64, 2, 128), device=DEV, dtype=BF16) for _ in range(2)]
    again = [x.clone() for x in pools]
    table, starts, cu, rot = i32([[3, 1], [0, 8]]), i32([5, 60]), i32([0, 40, 90]), PG.rotations(300, device=DEV)
    want = PG.append(*(x.contiguous() for x in qkv.split([8, 2, 2], 1)), *again, table, starts, cu, rot)
    q, k, v = qkv.split([8, 2, 2], 1)
    assert PG.append(q, k, v, *pools, table, starts, cu, rot, out=q) is q
    assert torch.equal(q, want) and all(torch.equal(a, b) for a, b in zip(pools, again))


@gpu
def test_append_many_requests():
    new = [i % 3 for i in range(5000)]
    tokens = sum(new)
    g = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randn((tokens, 1, 128), device=DEV, generator=g).to(F16) for _ in range(2))
    pools = [torch.zeros((5000, 64, 1, 128), device=DEV, dtype=F16) for _ in range(2)]
    table = torch.randperm(5000, device=DEV, generator=g).to(I32)[:, None]
    starts = torch.randint(0, 60, (5000,), device=DEV, generator=g).to(I32)
    PG.append(None, k, v, *pools, table, starts, offsets(new), PG.rotations(64, device=DEV))
    of = torch.tensor([r for r, n in enumerate(new) for _ in range(n)], device=DEV)
    at = starts[of].long() + torch.tensor([i for n in new for i in range(n)], device=DEV)
    assert torch.equal(pools[1][table[of, 0].long(), at], v)
    assert int((pools[1] != 0).any(-1).sum()) == tokens


@gpu
@pytest.mark.parametrize("counts", [[1], [3, 0, 5], [64, 65, 200], [256]])
@pytest.mark.parametrize("kv_heads,dtype,major", [(1, BF16, "token"), (3, F16, "head")])
def test_keep(counts, kv_heads, dtype, major):
    print("keep", counts, kv_heads, dtype, major, flush=True)
    g = torch.Generator(device=DEV).manual_seed(sum(counts))
    pages = 80
    shape = (pages, 64, kv_heads, 128) if major == "token" else (pages, kv_heads, 64, 128)
    pools = [torch.randn(shape, device=DEV, generator=g).to(dtype) for _ in range(2)]
    pools = [x if major == "token" else x.transpose(1, 2) for x in pools]
    want = [x.clone() for x in pools]
    table = torch.randperm(pages, device=DEV, generator=g)[:20 * len(counts)].view(-1, 20).to(I32)
    starts = [(61 * r + 5) % 200 for r in range(len(counts))]
    ids = []
    for n in counts:
        step = torch.randint(0, 4, (n,), device=DEV, generator=g)
        ids.append((torch.arange(n, device=DEV) + step.cumsum(0)).tolist())
    for pool in want:
        was = pool.clone()
        for r, mine in enumerate(ids):
            for i, j in enumerate(mine):
                a, b = starts[r] + i, starts[r] + j
                pool[int(table[r, a // 64]), a % 64] = was[int(table[r, b // 64]), b % 64]
    assert PG.keep(*pools, table, i32(starts), i32(sum(ids, [])), offsets(counts)) is None
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


@gpu
def test_keep_skips():
    """Ids below their index, negative starts, positions past the table, pages outside the pool."""
    pools = [torch.randn((6, 64, 2, 128), device=DEV).to(BF16) for _ in range(2)]
    want = [x.clone() for x in pools]
    table = i32([[0, 1], [2, 6], [3, 4], [5, -1]])
    for pool, was in zip(want, [x.clone() for x in pools]):
        pool[0, 11] = was[0, 14]      # request 0: [0, 4, 1, -3]: 4 moves; 1 and -3 lie below their index
    # request 1: its second page is not there; 2: a negative start; 3: past the table
    PG.keep(*pools, table, i32([10, 63, -1, 126]), i32([0, 4, 1, -3, 1, 2, 1, 5, 5, 5]), i32([0, 4, 6, 8, 10]))
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


@gpu
def test_rotations_table():
    rot = PG.rotations(100000, 64, 500000.0, device=DEV)
    at = torch.tensor([0, 1, 99999], device=DEV)
    angle = at.double()[:, None] * 500000.0 ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)
    assert rot.shape == (100000, 64) and rot.dtype == torch.float32
    assert torch.equal(rot[at], torch.cat([angle.cos(), angle.sin()], 1).float())
    with pytest.raises(ValueError, match="multiple of 16"):
        PG.rotations(10, 24)
