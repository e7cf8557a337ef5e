"""K / V pages of 16-bit numbers: the forms that large calls take, at sizes that the float64
reference can follow.  Which form a call takes follows from its sizes alone, here of 256 CUs:

  whole    work-groups of 256 columns, a request's keys in one part (more than 1024 work-groups)
  cut      the same over parts of the keys that are planned on the device (tables of more than 128
           entries, two requests of 80 work-groups)
  batch    blocks counted from cu_q on the device, where one request has most of the queries; of
           128 columns, and with many heads and wide tables of 256
  crowded  few queries of as many requests as half of the work-groups that run at once, the longer
           ones cut in two

Bounds as in test_gpu_paged.  A call with parts needs a workspace, which tells them apart."""
import math

import pytest
import torch

from conftest import pkg
from test_gpu_paged import (BF16, DEV, F16, I32, PG, check, chains, gen, make, offsets, random_tree, reference, rows_of,
                            seen_and_distance)

gpu = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def shared(g, lens, kv_heads, dtype, width):
    """Requests whose tables hold the same pages, each in an order of its own; -1 behind each request's pages."""
    pages = max(-(-n // 64) for n in lens) + 3
    pools = [torch.randn((pages, 64, kv_heads, 128), generator=g, device=DEV).to(dtype) for _ in range(2)]
    order = torch.randperm(pages, generator=g, device=DEV).to(I32)
    table = torch.full((len(lens), width), -1, dtype=I32, device=DEV)
    for r, n in enumerate(lens):
        need = -(-n // 64)
        table[r, :need] = order.roll(5 * r + 1)[:need]
    return pools, table


def widened(table, width):
    wide = torch.full((table.shape[0], max(width, table.shape[1])), -1, dtype=I32, device=DEV)
    wide[:, :table.shape[1]] = table
    return wide


def tree_seen(parents, n, window):
    """As seen_and_distance, of drafts behind a long context."""
    nq, paths = len(parents), chains(parents)
    before, context = n - nq, torch.arange(max(n - nq, 0))
    pos = torch.tensor([before + len(path) - 1 for path in paths])[:, None]
    own, away = torch.zeros((nq, nq), dtype=torch.bool), torch.zeros((nq, nq), dtype=torch.long)
    for i, path in enumerate(paths):
        own[i, path] = True
        away[i, path] = torch.arange(len(path))
    drop = max(-before, 0)  # (drafts that have no key)
    return (torch.cat([(context >= pos - window + 1) if window else torch.ones((nq, len(context)), dtype=torch.bool), own[:, drop:]], 1).to(DEV),
            torch.cat([(pos - context).abs(), away[:, drop:]], 1).to(DEV))


class Call:
    """A call of attend or attend_tree and what its rows should be."""

    def __init__(self, g, nq, lens, kv_heads, group, dtype, width=0, own_pages=True, lead=0, tail=0, most="given", tree=None, prefix=None,
                 document=None, slopes=False, cap=0.0, window=0):
        if own_pages:
            (self.kp, self.vp), table = make(g, lens, kv_heads, dtype)
            self.table = widened(table, width)
        else:
            (self.kp, self.vp), self.table = shared(g, lens, kv_heads, dtype, width)
        heads = kv_heads * group
        self.nq, self.lens, self.lead, self.tail, self.window, self.cap, self.tree = nq, lens, lead, tail, window, cap, tree
        self.kv_heads, self.group = kv_heads, group
        self.tokens = lead + sum(nq) + tail
        self.most = {"given": max(nq), None: None}.get(most, most)
        self.q = torch.randn((self.tokens, heads, 128), generator=g, device=DEV).mul_(1.5).to(dtype)
        self.q[:lead] = math.nan
        self.q[self.tokens - tail:] = math.nan
        self.cu, self.of_lens = offsets(nq) + lead, i32(lens)
        self.slopes = torch.exp2(-torch.arange(1, heads + 1, device=DEV) * 8.0 / heads).float() if slopes else None
        self.prefix, self.document = prefix, document
        self.more = dict(softcap=cap, slopes=self.slopes, window=window, return_lse=True)
        if tree is not None:
            self.parents = torch.full((self.tokens,), 7, dtype=I32, device=DEV)
            self.parents[lead:lead + sum(nq)] = i32(sum(tree, []))
        else:
            self.of_prefix = None if prefix is None else i32(prefix)
            self.of_document = None
            if document is not None:
                self.of_document = torch.zeros(self.tokens, dtype=I32, device=DEV)
                self.of_document[lead:lead + sum(nq)] = torch.cat(document).to(I32).to(DEV)

    def has_parts(self):
        most = self.tokens if self.most is None else min(self.most, self.tokens)
        return pkg("_lib").lib().v1_paged_attend_workspace(self.tokens, len(self.nq), self.kv_heads, self.group, most, 64 * self.table.shape[1],
                                                           self.window) > 0

    def __call__(self, out=None):
        args = self.q, self.kp, self.vp, self.table, self.of_lens
        if self.tree is not None:
            return PG.attend_tree(*args, self.parents, self.cu, self.most, out=out, **self.more)
        return PG.attend(*args, self.cu, self.most, prefix=self.of_prefix, document=self.of_document, out=out, **self.more)

    def requests(self):
        """Each request's rows of the output, keys, values, and what its queries see."""
        at = self.lead
        for r, n in enumerate(self.nq):
            first = n if self.most is None else min(n, self.most)
            if n:
                if self.tree is not None:
                    seen, away = tree_seen(self.tree[r], self.lens[r], self.window)
                else:
                    seen, away = seen_and_distance(n, self.lens[r], self.window, 0 if self.prefix is None else self.prefix[r],
                                                   None if self.document is None else self.document[r])
                yield (slice(at, at + first), slice(at + first, at + n), rows_of(self.kp, self.table[r], self.lens[r]),
                       rows_of(self.vp, self.table[r], self.lens[r]), seen[:first], away[:first])
            at += n

    def run_and_check(self, every=1):
        out, lse = self(torch.full_like(self.q, 123.0))
        for i, (mine, rest, k, v, seen, away) in enumerate(self.requests()):
            if i % every == 0:
                check(out[mine], lse[mine], self.q[mine], k, v, seen, away, cap=self.cap, slopes=self.slopes)
            assert bool((out[rest] == 123).all())
        assert bool((out[:self.lead] == 123).all()) and bool((out[self.tokens - self.tail:] == 123).all())
        again, same = self(torch.full_like(self.q, 123.0))
        assert torch.equal(out, again)
        for mine, *_ in self.requests():
            assert torch.equal(lse[mine], same[mine])


def documents(nq, lens, length=37):
    """Documents of `length` positions; one query's begins behind it."""
    of = [torch.arange(m - n, m) // length * length for n, m in zip(nq, lens)]
    of[0][5] = 10 ** 6
    return of


SCORES = [dict(), dict(cap=50.0), dict(cap=1.0), dict(slopes=True), dict(cap=5.0, slopes=True)]


# -------------------------------------------------------- 256 columns, one part
@gpu
@pytest.mark.parametrize("more", SCORES + [dict(window=100, prefix=[70, 3]), dict(document=True, prefix=[10, 500]),
                                           dict(window=37, slopes=True, cap=30.0, prefix=[150, 0]), dict(document=True, cap=30.0, window=20)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_whole(more, dtype):
    print("whole", more, dtype, flush=True)
    nq, lens = [700, 400], [900, 401]
    if "document" in more:
        more = {**more, "document": documents(nq, lens)}
    call = Call(gen(61), nq, lens, 32, 4, dtype, most=None, **more)   # 2 x 18 blocks x 32 KV heads
    assert not call.has_parts()
    call.run_and_check()


@gpu
@pytest.mark.parametrize("more", SCORES + [dict(window=30), dict(window=70, cap=40.0, slopes=True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_whole_trees(more, dtype):
    print("whole trees", more, dtype, flush=True)
    nq = [100, 3, 65, 0] * 10
    before = [(91 * i) % 400 for i in range(40)]
    call = Call(gen(62), nq, [a + b for a, b in zip(nq, before)], 8, 8, dtype, width=10, own_pages=False,
                tree=[random_tree(n, 7 * i + n, 1 + i % 3) for i, n in enumerate(nq)], **more)   # 40 x 4 blocks x 8 KV heads
    assert not call.has_parts()
    call.run_and_check(every=4)


# ----------------------------------------------------------- 256 columns, parts
@gpu
@pytest.mark.parametrize("more", SCORES + [dict(window=8400, prefix=[70, 3]), dict(document=True, prefix=[5000, 10]),
                                           dict(window=8300, cap=30.0, slopes=True, prefix=[150, 0])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cut(more, dtype):
    print("cut", more, dtype, flush=True)
    nq, lens = [300, 200], [9050, 3000]
    if "document" in more:
        more = {**more, "document": documents(nq, lens, 3700)}
    call = Call(gen(63), nq, lens, 8, 8, dtype, **more)   # 2 x 10 blocks x 8 KV heads
    assert call.has_parts()
    call.run_and_check()


@gpu
@pytest.mark.parametrize("more", SCORES + [dict(window=8300), dict(window=8250, cap=40.0, slopes=True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cut_trees(more, dtype):
    print("cut trees", more, dtype, flush=True)
    nq = [64, 33, 1, 0] * 4
    before = [0, 9000, 100, 64, 4000, 63, 8700, 1] * 2
    call = Call(gen(64), nq, [a + b for a, b in zip(nq, before)], 4, 8, dtype, width=145, own_pages=False,
                tree=[random_tree(n, 7 * i + n, 1 + i % 3) for i, n in enumerate(nq)], **more)   # 16 x 2 blocks x 4 KV heads
    assert call.has_parts()
    call.run_and_check()


# ------------------------------------------------- blocks counted on the device
@gpu
@pytest.mark.parametrize("more", SCORES + [dict(window=50, prefix=True), dict(document=True, prefix=True), dict(window=20, cap=30.0, slopes=True)])
@pytest.mark.parametrize("kv_heads,group,width,dtype", [(1, 4, 0, BF16), (4, 8, 150, F16), (4, 8, 150, BF16), (1, 5, 0, F16)])
def test_batch(more, kv_heads, group, width, dtype):
    """A chunk of 300 tokens, nineteen single tokens and requests without any; the first 250 of the chunk alone."""
    print("batch", more, kv_heads, group, width, dtype, flush=True)
    nq = [1] * 7 + [300] + [1] * 12 + [0, 2, 0]
    lens = [(71 * i) % 300 + 2 for i in range(len(nq))]
    lens[7], lens[3] = 420, 1
    if "window" in more and width:
        more = {**more, "window": 8200 + more["window"]}
    if "prefix" in more:
        more = {**more, "prefix": [(13 * i) % 90 for i in range(len(nq))]}
    if "document" in more:
        doc = [torch.arange(m - n, m) // 37 * 37 for n, m in zip(nq, lens)]
        doc[7][5] = 10 ** 6
        more = {**more, "document": doc}
    for most in ("given", 250):
        call = Call(gen(65), nq, lens, kv_heads, group, dtype, width=width, lead=5, tail=9, most=most, **more)
        assert not call.has_parts()
        call.run_and_check()


@gpu
@pytest.mark.parametrize("more", [dict(), dict(cap=3.0, slopes=True), dict(window=40)])
@pytest.mark.parametrize("kv_heads,group,width,dtype", [(2, 8, 0, F16), (4, 16, 150, BF16)])
def test_batch_of_trees(more, kv_heads, group, width, dtype):
    print("batch of trees", more, kv_heads, group, width, dtype, flush=True)
    nq = [1] * 8 + [200] + [3] * 9 + [0, 2]
    lens = [n + (71 * i) % 300 for i, n in enumerate(nq)]
    if "window" in more and width:
        more = dict(window=8240)
    call = Call(gen(66), nq, lens, kv_heads, group, dtype, width=width, lead=3, tail=4, tree=[random_tree(n, i + n) for i, n in enumerate(nq)], **more)
    assert not call.has_parts()
    call.run_and_check()


@gpu
def test_batch_of_300_requests():
    """More requests than a wave looks at in one go and than the plan by lengths takes."""
    nq = [600 if i == 170 else i % 3 * (i % 7 > 2) for i in range(300)]
    lens = [n + (37 * i) % 200 for i, n in enumerate(nq)]
    for most in ("given", None):
        Call(gen(67), nq, lens, 1, 2, BF16, width=13, own_pages=False, most=most, lead=2, tail=2).run_and_check()


# ------------------------------------------------ few queries of many requests
@gpu
@pytest.mark.parametrize("requests,kv_heads,group,most,longest,more", [
    (70, 8, 4, 1, 9000, dict()), (130, 1, 4, 1, 20000, dict()), (40, 32, 2, 1, 9000, dict()), (70, 8, 3, 1, 7000, dict(cap=2.0)),
    (150, 2, 6, 1, 9000, dict(slopes=True)), (200, 1, 16, 1, 12000, dict(cap=30.0, slopes=True)), (70, 8, 7, 4, 6000, dict()),
    (130, 1, 8, 4, 12000, dict(tree=True)), (70, 8, 2, 3, 6000, dict(prefix=True, document=True))])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_crowded(requests, kv_heads, group, most, longest, more, dtype):
    """Contexts from none to the longest; the long ones in two parts, the others in one."""
    print("crowded", requests, kv_heads, group, most, longest, more, dtype, flush=True)
    g = gen(68)
    nq = [1 + i % most for i in range(requests)]
    lens = [int(longest * ((i * 37) % requests / (requests - 1)) ** 2) for i in range(requests)]
    lens[3], lens[5], lens[6] = longest, longest - 63, 65
    if "tree" in more:
        lens = [max(n, m) for n, m in zip(nq, lens)]
        more = dict(tree=[random_tree(n, i) for i, n in enumerate(nq)])
    if "document" in more:
        more = dict(prefix=[(13 * i) % 90 for i in range(requests)], document=[torch.full((n,), m // 2) for n, m in zip(nq, lens)])
    call = Call(g, nq, lens, kv_heads, group, dtype, width=-(-longest // 64) + 1, own_pages=False, most=most, **more)
    assert call.has_parts()
    call.run_and_check()


@gpu
@pytest.mark.parametrize("nq,prefix", [(1, [4, 4096, 6001, 0]), (6, [6001, 100, 5999, 3]), (40, [4096, 6001, 1, 2500])])
def test_a_long_prefix_beside_a_short_window(nq, prefix):
    print("long prefix", nq, prefix, flush=True)
    Call(gen(69), [nq] * 4, [6001, 5000, 6000, 2000], 2, 4, BF16, window=64, prefix=prefix).run_and_check()


# -------------------------------------------- infinities and NaN that are masked
FORMS = {
    "whole": dict(nq=[700, 400], lens=[900, 401], kv_heads=32, group=4, most=None),
    "cut": dict(nq=[300, 200], lens=[9050, 3000], kv_heads=8, group=8),
    "batch": dict(nq=[1] * 7 + [300] + [1] * 12, lens=[50 + i for i in range(7)] + [4000] + [90 + i for i in range(12)], kv_heads=1, group=4),
    "wide batch": dict(nq=[1] * 7 + [300] + [1] * 12, lens=[50 + i for i in range(7)] + [2000] + [90 + i for i in range(12)], kv_heads=4, group=8, width=150),
    "small blocks": dict(nq=[40, 60], lens=[5000, 700], kv_heads=1, group=4),
    "few": dict(nq=[5, 3], lens=[5000, 700], kv_heads=2, group=5),
}


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("more", [dict(), dict(slopes=True), dict(cap=20.0), dict(cap=20.0, slopes=True), dict(window=90, prefix=True)])
@pytest.mark.parametrize("odd", [math.inf, math.nan])
def test_odd_values(form, more, odd):
    """Infinite and NaN values of keys in the middle of a request's queries, and of two before them: queries that do not see
    them are as if they were zero, columns of ones that do are infinite or NaN, their other columns as ever."""
    print("odd", form, more, odd, flush=True)
    how = FORMS[form]
    if "prefix" in more:
        more = dict(window=90, prefix=[20] * len(how["nq"]))
    dtype = F16 if math.isnan(odd) else BF16
    call = Call(gen(70), dtype=dtype, **how, **more)
    big = max(range(len(how["nq"])), key=lambda r: how["nq"][r])
    n, nq = how["lens"][big], how["nq"][big]
    places = {n - 1 - nq // 2: 5, n - nq - 1: 77, 30: 100}  # (position: column)
    keep = [c for c in range(128) if c not in places.values()]
    for at, col in places.items():
        call.vp[call.table[big, at // 64].long(), at % 64, :, col] = odd
    out, lse = call()
    for r, (mine, _, k, v, seen, away) in enumerate(call.requests()):
        got, plain = out[mine].clone(), torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
        if r == big:
            for at, col in places.items():
                sees = seen[:, at]
                x = got[sees][..., col]
                # (0 inf is NaN where a distance leaves the key a probability below fp32's)
                assert bool((torch.isnan(x) if math.isnan(odd) else ~torch.isfinite(x) if call.slopes is not None else x == odd).all()), (at, col)
                without = ~sees
                if bool(without.any()):
                    check(got[without][..., col:col + 1], lse[mine][without], call.q[mine][without], k, plain[..., col:col + 1], seen[without],
                          away[without], cap=call.cap, slopes=call.slopes)
            got, plain = got[..., keep], plain[..., keep]
        check(got, lse[mine], call.q[mine], k, plain, seen, away, cap=call.cap, slopes=call.slopes)


@gpu
@pytest.mark.parametrize("form", ["whole", "cut"])
@pytest.mark.parametrize("more", [dict(), dict(slopes=True, cap=4.0)])
def test_odd_values_in_trees(form, more):
    """An infinite value of a draft reaches its descendants alone, and a NaN key of one."""
    print("odd trees", form, more, flush=True)
    g = gen(71)
    if form == "whole":
        nq, before, kv_heads, group, width = [100] * 20 + [2] * 20, [30] * 40, 8, 8, 10
    else:
        nq, before, kv_heads, group, width = [64, 33, 1, 5] * 4, [9000, 300, 64, 7] * 4, 4, 8, 145
    tree = [random_tree(n, i) for i, n in enumerate(nq)]
    call = Call(g, nq, [a + b for a, b in zip(nq, before)], kv_heads, group, BF16, width=width, tree=tree, **more)
    assert call.has_parts() == (form == "cut")
    draft = 20
    page, row = call.table[0, (before[0] + draft) // 64].long(), (before[0] + draft) % 64
    call.vp[page, row, :, 9] = -math.inf
    out, lse = call()
    sees = torch.tensor([draft in path for path in chains(tree[0])], device=DEV)
    mine, _, k, v, seen, away = next(call.requests())
    v = v.masked_fill(torch.isinf(v), 0.0)
    assert 1 < int(sees.sum()) < nq[0] and bool((out[mine][sees][..., 9] == -math.inf).all())
    got = out[mine].clone()
    check(got[~sees], lse[mine][~sees], call.q[mine][~sees], k, v, seen[~sees], away[~sees], cap=call.cap, slopes=call.slopes)
    check(got[sees][..., 10:], lse[mine][sees], call.q[mine][sees], k, v[..., 10:], seen[sees], away[sees], cap=call.cap, slopes=call.slopes)
    call.vp[page, row, :, 9] = 0.0
    call.kp[page, row] = math.nan
    out, lse = call()
    assert bool(torch.isnan(out[mine][sees]).all()) and bool(torch.isnan(lse[mine][sees]).all())
    check(out[mine][~sees], lse[mine][~sees], call.q[mine][~sees], k.nan_to_num(0.0), v, seen[~sees], away[~sees], cap=call.cap, slopes=call.slopes)


@gpu
@pytest.mark.parametrize("form", ["whole", "cut", "batch", "wide batch"])
@pytest.mark.parametrize("more", [dict(), dict(slopes=True)])
def test_pages_that_are_not_there(form, more):
    print("missing pages", form, more, flush=True)
    call = Call(gen(72), dtype=BF16, **FORMS[form], **more)
    big = max(range(len(call.nq)), key=lambda r: call.nq[r])
    gone = {1: -1, 4: call.kp.shape[0], call.lens[big] // 64: 1 << 30}
    clean = call.table.clone()
    for entry, page in gone.items():
        call.table[big, entry] = page
    out, lse = call()
    call.table = clean
    for r, (mine, _, k, v, seen, away) in enumerate(call.requests()):
        if r == big:
            at = torch.arange(call.lens[big], device=DEV) // 64
            for entry in gone:
                seen = seen & (at != entry)
        check(out[mine], lse[mine], call.q[mine], k, v, seen, away, slopes=call.slopes)


# ---------------------------------------------------------- captured and replayed
@gpu
@pytest.mark.parametrize("form", ["cut", "batch", "wide batch"])
def test_captured_with_lengths_that_change(form):
    """Lengths and the requests' bounds change between the replays; each equals the eager call."""
    print("captured", form, flush=True)
    how = FORMS[form]
    call = Call(gen(73), dtype=BF16, cap=10.0, lead=4, tail=6, **how)
    for pool in (call.kp, call.vp):
        pool.nan_to_num_(0.0)
    call.table.clamp_(min=0)
    call.q.nan_to_num_(0.0)
    room = 64 * call.table.shape[1]
    out, graph = torch.zeros_like(call.q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = call(out)
    for replay in range(4):
        counts = list(how["nq"])
        counts = counts[replay:] + counts[:replay]
        call.cu.copy_(offsets(counts) + replay)
        call.of_lens.copy_(torch.randint(0, room, (len(counts),), device=DEV, generator=gen(replay), dtype=I32))
        want = torch.full_like(call.q, 9.0)
        out.fill_(9.0)
        _, want_lse = call(want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mine = slice(replay, replay + sum(counts))
        assert torch.equal(out, want) and torch.equal(lse[mine], want_lse[mine]), replay


# --------------------------------------------------------- two numbers a probability
# A request of at most 32 columns: a probability is two numbers of the type, whose rest is u^2 of it (fp16 at most 2^-25
# where the largest is 2^7 or more), so that beside the output's rounding there are the sums' errors alone,
#   |out - ref| <= u |ref| (1 + u) + A (u^2 + 2^-21 + 2 n 2^-24 + 2 d) + [fp16] n 2^-31 max |v|
# (n fp32 additions of a product and of the total at most; exponential, reciprocal and the last product 2^-21).
def two_groups(dtype, n):
    """Keys that score 0 and -c in turn, where the rounding of exp(-c) to the type is near half a step, and values of two
    signs that nearly cancel: keys [n], values [n], float64."""
    u = torch.finfo(dtype).eps / 2
    c = torch.arange(8, 120, dtype=torch.float64) / 64
    p = torch.exp(-c)
    off = (p.to(dtype).double() - p) / p
    c = c[off.abs().argmax()]
    assert float(off.abs().max()) > 0.4 * u
    second = torch.arange(n) % 2 == 1
    return torch.where(second, -c, torch.zeros(())), torch.where(second, torch.exp(c), torch.tensor(-1.0, dtype=torch.float64)).to(dtype).double()


def bound_of_two(ref, mag, n, d, most, dtype):
    u = torch.finfo(dtype).eps / 2
    return u * ref.abs() * (1 + u) + mag * (u * u + 2.0 ** -21 + 2 * n * 2.0 ** -24 + 2 * d) + (n * 2.0 ** -31 * most if dtype == F16 else 0.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_number_a_probability_would_not_pass(dtype):
    """The bound tells them apart: probabilities that are rounded once, totals that are not."""
    n = 640
    score, v = two_groups(dtype, n)
    p = torch.exp(score)
    ref, mag, once = (p @ v) / p.sum(), (p @ v.abs()) / p.sum(), (p.to(dtype).double() @ v) / p.sum()
    bound = bound_of_two(ref, mag, n, 0.0, v.abs().max(), dtype)
    assert float((once - ref).abs()) > float(bound)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("requests,nq,kv_heads,group", [(1, 1, 1, 4), (3, 1, 4, 8), (2, 4, 2, 8), (2, 2, 1, 5), (140, 1, 4, 4)])
def test_two_numbers_a_probability(dtype, requests, nq, kv_heads, group):
    print("two numbers", dtype, requests, nq, kv_heads, group, flush=True)
    n = 640
    score, v = two_groups(dtype, n)
    kp, vp = (torch.zeros((11, 64, kv_heads, 128), device=DEV, dtype=dtype) for _ in range(2))
    kp[:10, :, :, 0] = score.view(10, 64, 1).to(DEV).to(dtype)
    vp[:10] = v.view(10, 64, 1, 1).to(DEV).to(dtype)
    q = torch.zeros((requests * nq, kv_heads * group, 128), device=DEV, dtype=dtype)
    q[..., 0] = 1.0
    table = torch.arange(10, device=DEV, dtype=I32).expand(requests, 10)
    out, lse = PG.attend(q, kp, vp, table, i32([n] * requests), offsets([nq] * requests), nq, softmax_scale=1.0, return_lse=True)
    seen, away = seen_and_distance(nq, n)
    ref, mag, ref_lse, d, most = reference(q[:nq], rows_of(kp, table[0], n), rows_of(vp, table[0], n), seen, away, 1.0)
    bound = bound_of_two(ref, mag, n, d[..., None], most[None, :, None], dtype)
    off = (out.double().view(requests, nq, -1, 128) - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
