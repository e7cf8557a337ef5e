"""Calls of the attention over latent rows and 8-bit pages, and of their writers, that
the library refuses before it launches anything."""
import pytest

from conftest import pkg


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
