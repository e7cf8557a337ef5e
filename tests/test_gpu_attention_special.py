"""Scores that overflow to -inf: a key whose score is -inf weighs nothing beside
finite ones, and where all of a row's scores are -inf the softmax is 0 / 0, NaN with
a log-sum-exp of -inf, however its keys are split; a row without keys gives zeros."""
import math

import pytest
import torch

import test_gpu_expanded as expanded
import test_gpu_kv8 as kv8
import test_gpu_latent as latent
from conftest import pkg

LT, K8 = pkg("latent"), pkg("kv8")
DEV = "cuda:0"
gpu = pytest.mark.gpu
I32 = torch.int32


def undefined(out, lse):
    return bool(out.isnan().all()) and bool((lse == -math.inf).all())


def nothing(out, lse):
    return bool((out == 0).all()) and bool((lse == -math.inf).all())


@gpu
@pytest.mark.parametrize("rows,heads", [(6, 16), (6, 64), (300, 16), (300, 40)])  # (parts; one part)
@pytest.mark.parametrize("ragged", [False, True])
def test_latent(rows, heads, ragged):
    print("latent -inf", rows, heads, ragged, flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows + heads)
    pool, q = latent.rand_pool(g, 2000), latent.rand_q(g, rows, heads)
    rope = torch.zeros((2000, 64), device=DEV, dtype=torch.bfloat16)
    rope[:1000, 0] = 2.0 ** 100  # rows below 1000: -inf for the queries below
    pool[:, 512:640] = rope.view(torch.uint8)
    q[:, :, 512] = -(2.0 ** 100)
    keys = 900
    ids = torch.randint(0, 1000, (rows, keys), device=DEV, generator=g, dtype=I32)
    ids[1::6, 777] = 1500                                  # one finite key
    ids[2::6, ::2] += 1000                                 # every other
    ids[3::6] = -1                                         # none
    ids[4::6, 1:] = -1                                     # one key, -inf
    lens = torch.full((rows,), keys, device=DEV, dtype=I32) if ragged else None
    if ragged:
        lens[5::6] = 65
    out, lse = LT.attend(q, pool, ids, lens=lens, return_lse=True)
    for r in range(rows):
        if r % 6 in (0, 4, 5):
            assert undefined(out[r], lse[r]), r
        elif r % 6 == 3:
            assert nothing(out[r], lse[r]), r
    some = [r for r in range(rows) if r % 6 in (1, 2)][:20]
    latent.check(out[some], lse[some], q[some], pool, [ids[r][ids[r] >= 1000] for r in some], 192 ** -0.5)


@gpu
@pytest.mark.parametrize("rows,heads", [(6, 1), (6, 4), (600, 2)])
@pytest.mark.parametrize("ragged", [False, True])
def test_kv8(rows, heads, ragged):
    print("kv8 -inf", rows, heads, ragged, flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows + heads)
    (kp, ks), (vp, vs) = kv8.rand_pool(g, 40, heads), kv8.rand_pool(g, 40, heads)
    kp.view(torch.uint8)[:, :, :, 0] = 0
    kp[:20, :, :, 0] = 448.0  # pages below 20: -inf for the queries below
    pools = [kp, vp, ks, vs]
    q = torch.randn((rows, 4 * heads, 128), device=DEV, generator=g).to(torch.bfloat16)
    q[:, :, 0] = -(2.0 ** 127)
    keys = 900
    table = torch.arange(40, device=DEV, dtype=I32)
    ids = torch.randint(0, 1280, (rows, keys), device=DEV, generator=g, dtype=I32)
    ids[1::6, 777] = 1500
    ids[2::6, ::2] += 1280
    ids[3::6] = -1
    ids[4::6, 1:] = -1
    lens = torch.full((rows,), keys, device=DEV, dtype=I32) if ragged else None
    if ragged:
        lens[5::6] = 65
    out, lse = K8.attend(q, *pools, table, lens, ids, return_lse=True)
    for r in range(rows):
        if r % 6 in (0, 4, 5):
            assert undefined(out[r], lse[r]), r
        elif r % 6 == 3:
            assert nothing(out[r], lse[r]), r
    some = [r for r in range(rows) if r % 6 in (1, 2)][:20]
    kv8.check(out[some], lse[some], q[some], pools, [kv8.keys_of(table, ids[r][ids[r] >= 1280], keys, 40) for r in some])


@gpu
@pytest.mark.parametrize("heads,nq,nk", [(2, [100], [3000]), (300, [100], [300]), (1, [300, 5], [3000, 900])])  # (parts; one part; parts)
def test_expanded(heads, nq, nk):
    print("expanded -inf", heads, nq, flush=True)
    q, kv, rope, cu_q, cu_k = expanded.inputs(heads, nq, nk, heads)
    q[..., 0] = -(2.0 ** 100)
    kv[..., 0] = 2.0 ** 100
    out, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max(nq), return_lse=True)
    assert undefined(out, lse)
    for j in [200] + ([3000 + 850] if len(nk) > 1 else []):  # one finite key of each sequence, which every query sees
        kv[j, :, 0] = 0
    out, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, max(nq), return_lse=True)
    for b, j in enumerate([200, 3000 + 850][:len(nq)]):
        i, n = int(cu_q[b]), nq[b]
        for h in range(0, heads, 37):
            expanded.check(out[i:i + n, h:h + 1], lse[i:i + n, h:h + 1], q[i:i + n, h:h + 1], kv[j:j + 1, h:h + 1], rope[j:j + 1], [n], [1], False)
    none = torch.zeros_like(cu_k)
    assert nothing(*LT.attend_expanded(q, kv, rope, cu_q, none, max(nq), return_lse=True))
