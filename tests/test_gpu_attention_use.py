"""The 8-bit and latent caches and their attention as programs use them: captured
into graphs and replayed over new contents, on streams and threads of their own,
with padded rows, short lengths in tables of 2^30 positions, and queries behind
max_q.  A result is compared with the same call's made alone (no operator's order
of sums depends on timing, so they are equal), or with the checks of the
operators' own tests."""
import contextlib
import importlib
import math
import re
import struct
import threading
from pathlib import Path

import pytest
import torch

import test_gpu_expanded as expanded
import test_gpu_kv8 as kv8
import test_gpu_latent as latent
from conftest import pkg

LT, K8 = pkg("latent"), pkg("kv8")
DEV = "cuda:0"
gpu = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32


class Use:
    """One call over tensors of its own: `refill` gives them new contents, `run`
    calls and returns every tensor that the call writes."""

    def __init__(self, kind, seed):
        self.kind, self.g = kind, torch.Generator(device=DEV).manual_seed(seed)
        self.t = {n: v.clone() for n, v in self.new().items()}

    def normal(self, *shape):
        return torch.randn(shape, device=DEV, generator=self.g).to(BF16)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=self.g, dtype=I32)

    def new(self):
        if self.kind == "latent_store":
            return dict(latent=self.normal(37, 512), rope=self.normal(37, 64), pool=torch.zeros((64, 656), device=DEV, dtype=torch.uint8),
                        slots=torch.randperm(64, device=DEV, generator=self.g)[:37].to(I32))
        if self.kind.startswith("latent"):  # one part of each row's keys, or several
            rows, heads, entries = (300, 16, 2) if self.kind == "latent" else (5, 24, 60)
            return dict(q=self.normal(rows, heads, 576), pool=latent.rand_pool(self.g, 4096), table=self.ints(0, 64, rows, entries),
                        lens=self.ints(0, 64 * entries + 1, rows))
        if self.kind.startswith("expanded"):
            n, heads = (300, 300) if self.kind == "expanded" else (700, 2)
            cut = int(self.ints(1, n, 1))
            return dict(q=self.normal(n, heads, 192), kv=self.normal(n, heads, 256), k_rope=self.normal(n, 64),
                        cu_q=torch.tensor([0, cut, n], device=DEV, dtype=I32))
        heads, rows = 2, 6
        (kp, ks), (vp, vs) = kv8.rand_pool(self.g, 64, heads), kv8.rand_pool(self.g, 64, heads)
        pools = dict(k_pool=kp, v_pool=vp, k_scale=ks, v_scale=vs)
        if self.kind == "kv8_store":
            cu = torch.cat([torch.zeros(1, device=DEV, dtype=I32), self.ints(0, 90, rows).cumsum(0).to(I32)])
            return dict(k=self.normal(540, heads, 128), v=self.normal(540, heads, 128), **pools, starts=self.ints(0, 300, rows),
                        table=torch.randperm(64, device=DEV, generator=self.g)[:60].to(I32).view(rows, 10), cu_tokens=cu)
        rows, entries = (520, 1) if self.kind == "kv8" else (rows, 40)
        return dict(q=self.normal(rows, heads * 4, 128), **pools, table=self.ints(0, 64, rows, entries),
                    lens=self.ints(0, 64 * entries + 1, rows))

    def refill(self):
        for name, v in self.new().items():
            self.t[name].copy_(v)

    def run(self):
        t = self.t
        if self.kind == "latent_store":
            LT.store_rows(**t)
            return [t["pool"]]
        if self.kind.startswith("latent"):
            return list(LT.attend(**t, page_bits=6, return_lse=True))
        if self.kind.startswith("expanded"):
            return list(LT.attend_expanded(**t, return_lse=True))
        if self.kind == "kv8_store":
            K8.store(**t)
            return [t[n].view(torch.uint8) if t[n].dtype == kv8.F8 else t[n] for n in ("k_pool", "v_pool", "k_scale", "v_scale")]
        return list(K8.attend(**t, return_lse=True))

    def alone(self):
        """What `run` gives for the present contents, which stay as they are."""
        saved = {n: v.clone() for n, v in self.t.items()}
        out = [x.clone() for x in self.run()]
        torch.cuda.synchronize()
        for n, v in saved.items():
            self.t[n].copy_(v)
        torch.cuda.synchronize()
        return out


KINDS = ["latent_store", "latent", "latent_parts", "expanded", "expanded_parts", "kv8_store", "kv8", "kv8_parts"]


def same(got, want):
    for a, b in zip(got, want):
        assert a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_graph_replays(kind):
    """Captured once, replayed over new contents, lengths and pages, with eager
    calls and work of other kinds between the replays."""
    print("graph", kind, flush=True)
    use = Use(kind, 1)
    use.alone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = use.run()
    for _ in range(4):
        use.refill()
        want = use.alone()
        torch.randn(1 << 20, device=DEV).sort()
        graph.replay()
        torch.cuda.synchronize()
        same(out, want)


@gpu
def test_two_graphs_of_one_stream_on_two_streams():
    print("two graphs", flush=True)
    stream = torch.cuda.Stream()
    uses, graphs, outs = [Use(k, s) for s in (2, 3) for k in ("latent_parts", "expanded_parts", "kv8_parts")], [], []
    wants = [u.alone() for u in uses]
    for half in (uses[:3], uses[3:]):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            outs += [u.run() for u in half]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            same(out, want)


@gpu
def test_threads_on_their_streams():
    print("threads", flush=True)
    uses = [Use(k, 4) for k in KINDS]
    wants = [u.alone() for u in uses]
    wrong = []

    def work(use, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    out = use.run()
                    if use.kind == "kv8_store":
                        break  # (it changes what it would start from)
                torch.cuda.current_stream().synchronize()
                same(out, want)
        except BaseException as e:  # noqa: B036 (handed to the test's own thread)
            wrong.append((use.kind, e))

    threads = [threading.Thread(target=work, args=a) for a in zip(uses, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_on_the_current_stream(kind):
    """The inputs are made, late, on the call's stream; nothing else orders the two."""
    print("stream", kind, flush=True)
    use = Use(kind, 5)
    late = {n: v.clone() for n, v in use.t.items()}
    want = use.alone()
    slow = torch.randn((4096, 4096), device=DEV)
    for v in use.t.values():
        v.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(10):
            slow = torch.tanh(slow @ slow)
        for n, v in late.items():
            use.t[n].copy_(v)
        out = use.run()
        torch.cuda.current_stream().synchronize()
        same(out, want)


@gpu
@pytest.mark.parametrize("rows,heads,keys", [(300, 4, 64), (2, 4, 3000)])
def test_padded_rows(rows, heads, keys):
    """Rows without keys are zeros and -inf whatever their queries hold."""
    print("padded", rows, keys, flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows)
    q = torch.full((rows, heads, 576), math.nan, device=DEV, dtype=BF16)
    pool = latent.rand_pool(g, 4096)
    none = torch.full((rows, keys), -1, device=DEV, dtype=I32)
    lens = torch.zeros(rows, device=DEV, dtype=I32)
    table = torch.arange((keys + 63) // 64, device=DEV, dtype=I32)
    (kp, ks), (vp, vs) = kv8.rand_pool(g, 64, 2), kv8.rand_pool(g, 64, 2)
    narrow = q[..., :128]
    for out, lse in (LT.attend(q, pool, none, return_lse=True), LT.attend(q, pool, table=table, page_bits=6, lens=lens, return_lse=True),
                     LT.attend(q, pool, none, lens=lens + keys, return_lse=True),
                     K8.attend(narrow, kp, vp, ks, vs, table, ids=none, return_lse=True),
                     K8.attend(narrow, kp, vp, ks, vs, table, lens, return_lse=True),
                     K8.attend(narrow, kp, vp, ks, vs, table, lens + keys, none, return_lse=True),
                     K8.attend(narrow, kp, vp, ks, vs, table - 64, return_lse=True)):
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    # queries before their sequence's keys begin, and a sequence without keys
    n = 300
    cu_q, cu_k = torch.tensor([0, n, n + 7], device=DEV, dtype=I32), torch.tensor([0, 5, 5], device=DEV, dtype=I32)
    q = torch.full((n + 7, heads, 192), math.nan, device=DEV, dtype=BF16)
    kv, rope = (torch.randn((5, *s), device=DEV, generator=g).to(BF16) for s in ((heads, 256), (64,)))
    out, lse = LT.attend_expanded(q, kv, rope, cu_q, cu_k, return_lse=True)
    none = torch.ones(n + 7, device=DEV, dtype=torch.bool)
    none[n - 5:n] = False
    assert bool((out[none] == 0).all()) and bool((lse[none] == -math.inf).all())
    assert bool(out[~none].isnan().all())


@gpu
@pytest.mark.parametrize("rows", [3, 200])
def test_short_rows_of_tables_of_2_30_positions(rows):
    """Capacities whose tiles, over all rows, are more than 32 bits can add."""
    print("long tables", rows, flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows)
    lens = torch.randint(0, 200, (rows,), device=DEV, generator=g, dtype=I32)
    lens[0], lens[1], lens[2] = 0, 1, 3000
    pool, q = latent.rand_pool(g, 3000), latent.rand_q(g, rows, 16)
    table = torch.zeros(1, device=DEV, dtype=I32)
    out, lse = LT.attend(q, pool, table=table, page_bits=30, lens=lens, return_lse=True)
    at = torch.arange(3000, device=DEV)
    latent.check(out, lse, q, pool, [at[:n] for n in lens.tolist()], 192 ** -0.5)
    (kp, ks), (vp, vs) = kv8.rand_pool(g, 64, 1), kv8.rand_pool(g, 64, 1)
    table = torch.randint(0, 64, (1 << 24,), device=DEV, generator=g, dtype=I32)
    q = torch.randn((rows, 4, 128), device=DEV, generator=g).to(BF16)
    out, lse = K8.attend(q, kp, vp, ks, vs, table, lens, return_lse=True)
    kv8.check(out, lse, q, [kp, vp, ks, vs], [kv8.keys_of(table, at, int(n), 64) for n in lens])


@gpu
def test_queries_behind_max_q():
    """A sequence longer than max_q: its first max_q queries are right, and what is
    not computed is left as it was (keys in one part, and in several)."""
    print("max_q", flush=True)
    for heads in (1, 300):
        q, kv, rope, cu = expanded.inputs(heads, [900], [900], heads)[:4]
        out = torch.full((900, heads, 128), 7.0, device=DEV, dtype=BF16)
        whole, whole_lse = LT.attend_expanded(q, kv, rope, cu, return_lse=True)
        _, lse = LT.attend_expanded(q, kv, rope, cu, max_q=100, out=out, return_lse=True)
        expanded.check(whole[:, :1], whole_lse[:, :1], q[:, :1], kv[:, :1], rope, [900], [900])
        # (each within u (|ref| + A) (1 + u) + 2 d A of the exact one, |ref| <= A <= the largest value, d < u / 8)
        close = (out.float() - whole.float()).abs() <= 5 * expanded.U * kv[:, :, 128:].float().abs().amax()
        assert bool(close[:100].all())
        assert bool((close | (out == 7)).flatten(1).all()) and bool((out[512:] == 7).all())


class _Entry:
    def __init__(self, calls):
        self.calls = calls

    def __call__(self, args, stream):
        self.calls.append((len(args), stream))
        return 0


def test_another_device_than_the_current_one(monkeypatch):
    """The call is made with the tensors' device current and on its stream."""
    L = importlib.import_module("10_20_amd._lib")
    calls, entered = [], []

    class Lib:
        v1_latent_store = _Entry(calls)

    class Tensor:
        def get_device(self):
            return 1

    @contextlib.contextmanager
    def device(index):
        entered.append(index)
        yield

    monkeypatch.setattr(L, "_lib", Lib())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    fields = [0] * len(L.PACKED["v1_latent_store"].unpack(bytes(L.PACKED["v1_latent_store"].size)))
    L.call_packed("v1_latent_store", Tensor(), *fields)
    assert entered == [1] and calls == [(L.PACKED["v1_latent_store"].size, 101)]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    L.call_packed("v1_latent_store", Tensor(), *fields)
    assert entered == [1] and len(calls) == 2


def test_too_many_positions():
    """Refused by the library itself, before any launch."""
    L = pkg("_lib")
    if not L.LIB_PATH.exists():
        pkg("build").build()
    h = L.lib()
    most = 2 ** 31 - 1
    for name, fields, text in (
            ("v1_latent_attend", [256, 576, 576, 256, 8, 656, 0, 0, 0, 256, 3, 0, 256, 512, 512, 0, 0, 0, 0, 1000, 1, most, 1.0], b"keys"),
            ("v1_kv8_attend", [256, 128, 128, 256, 8192, 128, 128, 256, 8192, 128, 128, 256, 1, 256, 1, 8, 256, 1, 0, 0, 0, 256, 128, 128,
                               0, 0, 0, 4, 1000, 1, 1, most, 1.0], b"keys"),
            ("v1_latent_expanded", [256, 192, 192, 256, 256, 256, 256, 64, 256, 256, 256, 128, 128, 0, 0, 0, 8, most, 1, 1, 8, 1, 1.0],
             b"keys")):
        assert getattr(h, name)(L.PACKED[name].pack(*fields), None) == L.V1_ERR_INVALID, name
        assert text in h.v1_last_error(), h.v1_last_error()


def test_argument_structures_match_the_header():
    """The packed formats hold the header's fields in its order, padded as C does."""
    L = pkg("_lib")
    text = re.sub(r"/\*.*?\*/", "", (Path(__file__).resolve().parents[1] / "include" / "v1idx.h").read_text(), flags=re.S)
    for name, packed in L.PACKED.items():
        body = re.search(r"typedef struct \{([^}]*)\} %s_args;" % name, text).group(1)
        want = ""
        for line in body.split(";"):
            kind = "q" if "*" in line or "int64_t" in line else "i" if "int32_t" in line else "f" if "float" in line else ""
            want += kind * (line.count(",") + 1) if kind else ""
        got = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([a-z])", packed.format) if c != "x")
        assert got == want, name
        assert packed.size == -(-struct.calcsize(want) // 8) * 8, name


@gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_nothing_to_attend(ragged):
    """Tables, pools and ids without an entry: rows of zeros and -inf."""
    print("nothing", ragged, flush=True)
    rows = 3
    q = torch.randn((rows, 4, 576), device=DEV).to(BF16)
    lens = torch.full((rows,), 5, device=DEV, dtype=I32) if ragged else None
    pool, none = torch.zeros((8, 656), device=DEV, dtype=torch.uint8), torch.zeros((rows, 0), device=DEV, dtype=I32)
    pools = lambda pages: (*(torch.zeros((pages, 64, 2, 128), device=DEV, dtype=torch.uint8).view(kv8.F8) for _ in range(2)),
                           *(torch.ones((pages, 2), device=DEV) for _ in range(2)))
    table = torch.zeros((rows, 2), device=DEV, dtype=I32)
    ids = torch.zeros((rows, 3), device=DEV, dtype=I32)
    narrow = q[..., :128].contiguous()
    for out, lse in (LT.attend(q, pool, none, lens=lens, return_lse=True), LT.attend(q, pool, table=none, page_bits=6, lens=lens, return_lse=True),
                     LT.attend(q, pool[:0], lens=lens, return_lse=True), LT.attend(q, pool[:0], ids, lens=lens, return_lse=True),
                     K8.attend(narrow, *pools(4), none, lens, return_lse=True), K8.attend(narrow, *pools(0), table, lens, return_lse=True),
                     K8.attend(narrow, *pools(4), table, lens, none, return_lse=True),
                     K8.attend(narrow, *pools(0), table, lens, ids, return_lse=True)):
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
