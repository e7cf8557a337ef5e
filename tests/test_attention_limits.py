"""Calls of the attention over latent rows and 8-bit pages, and of their writers, that
the library refuses before it launches anything."""
import importlib

import pytest
import torch

from conftest import pkg

LT, K8 = pkg("latent"), pkg("kv8")
BF16, F32, I32, F8 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn


def refused(name, **fields):
    L = pkg("_lib")
    if not L.LIB_PATH.exists():
        pkg("build").build()
    rc = getattr(L.lib(), name)(L.PACKED[name].pack(*fields.values()), None)
    return rc == L.V1_ERR_INVALID and L.lib().v1_last_error().decode()


ATTEND = dict(q=256, q_row=576, q_head=576, pool=256, pool_rows=8, stride=656, map=0, map_len=0, map_stride=0, ids=256, ids_stride=3, lens=0,
              out=256, o_row=512, o_head=512, lse=0, ws=0, ws_bytes=0, shift=0, rows=1000, heads=1, keys=3, scale=1.0)
STORE = dict(latent=256, ls=512, rope=256, rs=64, slots=256, pool=256, rows=8, stride=656, tokens=3)
KV8 = dict(q=256, qr=1024, qh=128, kp=256, kpp=8192, kpt=128, kph=128, vp=256, vpp=8192, vpt=128, vph=128, ks=256, ksp=1, vs=256, vsp=1,
           pages=4, table=256, ts=9, ids=0, ids_s=0, lens=0, out=256, o_row=512, o_head=128, lse=0, ws=0, wsb=0, tl=9, rows=4096, kv_heads=1,
           group=4, keys=100, scale=0.1)
KV8_STORE = dict(k=256, kt=128, kh=128, v=256, vt=128, vh=128, kp=256, kpp=8192, kpt=128, kph=128, vp=256, vpp=8192, vpt=128, vph=128, ks=256,
                 ksp=1, vs=256, vsp=1, pages=4, table=256, ts=9, starts=256, cu=256, tl=9, tokens=5, requests=2, kv_heads=1)


@pytest.mark.parametrize("name,fields,change", [
    ("v1_latent_attend", ATTEND, dict(rows=1 << 23)), ("v1_latent_attend", ATTEND, dict(rows=1 << 22, heads=128)),
    ("v1_latent_attend", ATTEND, dict(rows=(1 << 31) - 1)), ("v1_latent_store", STORE, dict(tokens=1 << 26)),
    ("v1_latent_store", STORE, dict(tokens=(1 << 31) - 1)), ("v1_kv8_attend", KV8, dict(rows=1 << 24)),
    ("v1_kv8_attend", KV8, dict(rows=1 << 22, kv_heads=16)), ("v1_kv8_attend", KV8, dict(rows=1 << 23, kv_heads=3)),
    ("v1_kv8_store", KV8_STORE, dict(tokens=1 << 25, requests=1 << 24)), ("v1_kv8_store", KV8_STORE, dict(tokens=(1 << 31) - 1))])
def test_more_work_groups_than_a_launch_holds(name, fields, change):
    """(A launch has fewer than 2^32 work-items a dimension.)"""
    assert "for a launch" in (refused(name, **{**fields, **change}) or ""), (name, change)


# ------------------------------------------------- arguments that do not fit are ValueErrors
@pytest.fixture
def on_meta(monkeypatch):
    """The modules' own checks, with tensors that have shapes and no memory; a call that
    reaches the library fails the test."""
    L = importlib.import_module("10_20_amd._lib")

    class Lib:
        def __getattr__(self, name):
            def entry(*args):
                raise AssertionError(f"{name} was called")
            return entry

    monkeypatch.setattr(L, "require_gpu", lambda *t: None)
    monkeypatch.setattr(L, "_lib", Lib())
    return lambda *shape, dtype=BF16: torch.empty(shape, device="meta", dtype=dtype)


def test_sizes_past_32_bits(on_meta):
    z, n = on_meta, 1 << 31
    pool = z(8, 656, dtype=torch.uint8)
    with pytest.raises(ValueError, match="2\\*\\*31"):
        LT.store_rows(z(n, 512), z(n, 64), pool, z(n, dtype=I32))
    for many in (n, 2 * n, 2 * n + 1):  # (the last: one key or row, if its low 32 bits were taken)
        for call in (lambda: LT.attend(z(many, 1, 576), pool, z(many, 3, dtype=I32), return_lse=True),
                     lambda: LT.attend(z(2, 1, 576), pool, z(2, many, dtype=I32)), lambda: LT.attend(z(2, many, 576), pool, z(2, 3, dtype=I32)),
                     lambda: LT.attend_expanded(z(many, 1, 192), z(5, 1, 256), z(5, 64), z(2, dtype=I32)),
                     lambda: LT.attend_expanded(z(5, 1, 192), z(many, 1, 256), z(many, 64), z(2, dtype=I32)),
                     lambda: LT.attend_expanded(z(5, 1, 192), z(5, 1, 256), z(5, 64), z(many + 1, dtype=I32))):
            with pytest.raises(ValueError, match="2\\*\\*31"):
                call()
        pools = z(3, 64, 1, 128, dtype=F8), z(3, 64, 1, 128, dtype=F8), z(3, 1, dtype=F32), z(3, 1, dtype=F32)
        for call in (lambda: K8.attend(z(2, 1, 128), *pools, z(2, 9, dtype=I32), ids=z(2, many, dtype=I32)),
                     lambda: K8.attend(z(many, 1, 128), *pools, z(9, dtype=I32)), lambda: K8.attend(z(2, 1, 128), *pools, z(many, dtype=I32)),
                     lambda: K8.store(z(many, 1, 128), z(many, 1, 128), *pools, z(2, 9, dtype=I32), z(2, dtype=I32), z(3, dtype=I32)),
                     lambda: K8.store(z(5, 1, 128), z(5, 1, 128), *pools, z(many, 9, dtype=I32), z(many, dtype=I32), z(many + 1, dtype=I32))):
            with pytest.raises(ValueError, match="2\\*\\*31"):
                call()


def test_dimensions_that_are_not_there(on_meta):
    z = on_meta
    pool = z(8, 656, dtype=torch.uint8)
    for latent, rope in ((z(), z(5, 64)), (z(512), z(5, 64)), (z(5, 512), z()), (z(5, 512), z(64)), (z(1, 5, 512), z(5, 64))):
        with pytest.raises(ValueError, match="must be"):
            LT.store_rows(latent, rope, pool, z(5, dtype=I32))
    for bad in (dict(kv=z()), dict(kv=z(5, 256)), dict(k_rope=z()), dict(k_rope=z(64)), dict(q=z()), dict(cu_q=z(dtype=I32)), dict(out=z())):
        with pytest.raises(ValueError, match="must be"):
            LT.attend_expanded(**{**dict(q=z(5, 1, 192), kv=z(5, 1, 256), k_rope=z(5, 64), cu_q=z(2, dtype=I32)), **bad})
    for bad in (dict(q=z()), dict(pool=z(dtype=torch.uint8)), dict(ids=z(dtype=I32)), dict(table=z(dtype=I32)), dict(lens=z(dtype=I32)), dict(out=z())):
        with pytest.raises(ValueError, match="must be"):
            LT.attend(**{**dict(q=z(5, 1, 576), pool=pool, ids=z(5, 3, dtype=I32)), **bad})
    codes, scales, table = z(3, 64, 1, 128, dtype=F8), z(3, 1, dtype=F32), z(2, 9, dtype=I32)
    base = dict(k_pool=codes, v_pool=codes, k_scale=scales, v_scale=scales, table=table)
    for bad in (dict(q=z()), dict(k_pool=z(dtype=F8)), dict(k_scale=z(dtype=F32)), dict(table=z(dtype=I32)), dict(lens=z(dtype=I32)),
                dict(ids=z(dtype=I32)), dict(out=z())):
        with pytest.raises(ValueError, match="must be"):
            K8.attend(**{**base, "q": z(2, 1, 128), **bad})
    for bad in (dict(k=z()), dict(table=z(dtype=I32)), dict(starts=z(dtype=I32)), dict(cu_tokens=z(dtype=I32)), dict(v_scale=z(dtype=F32))):
        with pytest.raises(ValueError, match="must be"):
            K8.store(**{**base, "k": z(5, 1, 128), "v": z(5, 1, 128), "starts": z(2, dtype=I32), "cu_tokens": z(3, dtype=I32), **bad})


def test_scales_that_the_library_refuses():
    expanded = dict(q=256, qr=384, qh=192, kv=256, kr=512, kh=256, rope=256, rr=64, cu_q=256, cu_k=256, out=256, o_row=256, o_head=128,
                    lse=0, ws=0, wsb=0, tokens=8, keys=8, batch=1, heads=1, max_q=8, causal=1, scale=0.1)
    for name, fields in (("v1_latent_attend", ATTEND), ("v1_kv8_attend", KV8), ("v1_latent_expanded", expanded)):
        for s in (3e38, 1e39, float("inf"), float("nan"), 0.0, 1e-60):  # (3e38 times log2(e) is no float32, 1e39 neither)
            assert "scale" in (refused(name, **{**fields, "scale": s}) or ""), (name, s)


@pytest.mark.parametrize("change", [dict(kp=264), dict(vp=8), dict(kpp=8200), dict(vpt=136), dict(kph=8)])
def test_pools_that_only_one_of_writer_and_reader_would_take(change):
    for name, fields in (("v1_kv8_store", KV8_STORE), ("v1_kv8_attend", KV8)):
        assert "pools must be 16-byte aligned" in (refused(name, **{**fields, **change}) or ""), name
