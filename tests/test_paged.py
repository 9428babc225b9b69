"""Paged-cache operators without a GPU: what the entry points refuse."""
import ctypes as C
import itertools
import re
import subprocess
from pathlib import Path

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from catopt_b200 import _lib, build

    build.build()
    return _lib.load()


P = 4096        # a non-null, aligned address; never read, every call here is refused before a launch

ATTEND = dict(q=P, qt=256, qh=64, k=P, v=P, ks=2 * 16 * 64, vs=2 * 16 * 64, o=2 * P, w=None, table=P, lens=P, cu=P, n=8, R=2, Hq=4,
              Hkv=2, d=64, page=16, n_pages=4, max_pages=2, max_q=4, max_k=32, scale=0.125, causal=1, dtype=1, scratch=P,
              bytes=1 << 30, status=None, stream=None)
APPEND = dict(q=P, qt=256, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, out=P, kp=P, vp=P, ks=2048, vs=2048, w=None, table=P,
              lens=P, cu=P, pos=P, qw=None, kw=None, eps=1e-6, cos=P, sin=P, rows=8, rot=64, inter=0, n=8, R=2, Hq=4, Hkv=2, d=64,
              page=16, n_pages=4, max_pages=2, dtype=1, status=None, stream=None)
EVICT = dict(k=P, v=P, ks=2048, vs=2048, w=P, table=P, lens=P, to=P, kept=P, new=P, R=2, Hkv=2, d=64, page=16, n_pages=4,
             max_pages=2, new_pages=1, max_k=32, budget=8, first=2, last=2, dtype=1, status=None, stream=None)
NULL, SHAPE, ALIGN, DTYPE, SCRATCH = 6, 1, 2, 3, 7


@pytest.mark.parametrize("change,want", [
    (dict(k=None), NULL), (dict(table=None), NULL), (dict(q=None), NULL), (dict(scratch=None), NULL), (dict(n=-1), SHAPE),
    (dict(R=0), SHAPE), (dict(Hq=3), SHAPE), (dict(Hkv=0), SHAPE), (dict(d=60), SHAPE), (dict(d=136), SHAPE), (dict(page=12), SHAPE),
    (dict(page=4), SHAPE), (dict(page=2048), SHAPE), (dict(max_k=33), SHAPE), (dict(max_k=0), SHAPE), (dict(max_q=-1), SHAPE),
    (dict(n_pages=0), SHAPE), (dict(scale=0.0), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(ks=2040), SHAPE), (dict(qt=0), SHAPE), (dict(o=P), SHAPE), (dict(qh=0), SHAPE), (dict(n=1 << 30), SHAPE), (dict(dtype=7), DTYPE), (dict(q=P + 2), ALIGN), (dict(qt=252), ALIGN),
    (dict(v=P + 8), ALIGN), (dict(w=P + 4), ALIGN), (dict(bytes=16), SCRATCH),
], ids=str)
def test_attention_refusals(lib, change, want):
    assert lib.cb2_om_paged_fwd(*{**ATTEND, **change}.values()) == want


@pytest.mark.parametrize("change,want", [
    (dict(k=None), NULL), (dict(out=None), NULL), (dict(cos=None), NULL), (dict(pos=None), NULL), (dict(cu=None), NULL),
    (dict(rot=66), SHAPE), (dict(rot=3), SHAPE), (dict(rows=0), SHAPE), (dict(d=4), SHAPE), (dict(page=17), SHAPE),
    (dict(eps=-1.0), SHAPE), (dict(eps=float("nan")), SHAPE), (dict(vs=8), SHAPE), (dict(n=-4), SHAPE), (dict(kt=-128), SHAPE),
    (dict(dtype=2), DTYPE), (dict(kt=130), ALIGN), (dict(vp=P + 4), ALIGN), (dict(qw=P + 2), ALIGN),
], ids=str)
def test_append_refusals(lib, change, want):
    assert lib.cb2_paged_append(*{**APPEND, **change}.values()) == want


@pytest.mark.parametrize("scale", [2.4e38, 3e38, 3.4e38])
def test_scale_in_base_two(lib, scale):
    # scale / ln 2 is what the kernels multiply by: it has to be finite
    assert lib.cb2_om_paged_fwd(*{**ATTEND, "scale": scale}.values()) == SHAPE


FAR = 1 << 20      # operands in places of their own, 8 rows of 4 (k, v: 2) heads of 64 bf16 each: 4096 (2048) bytes


@pytest.mark.parametrize("out", [FAR - 4080, FAR - 16, FAR + 16, FAR + 4080])
def test_attention_output_on_the_queries(lib, out):
    assert lib.cb2_om_paged_fwd(*{**ATTEND, "q": FAR, "o": out}.values()) == SHAPE
    # heads first in memory: rows of 512 bytes, 4 heads of 1024
    assert lib.cb2_om_paged_fwd(*{**ATTEND, "q": FAR, "qt": 64, "qh": 512, "o": out}.values()) == SHAPE


@pytest.mark.parametrize("change", [dict(out=FAR - 4080), dict(out=FAR + 16), dict(out=FAR + 4080),        # part of q
                                    dict(out=FAR, qt=512), dict(out=FAR, qt=64, qh=512),                    # q itself, not dense
                                    dict(out=2 * FAR - 4080), dict(out=2 * FAR + 2032), dict(out=3 * FAR - 16), dict(out=3 * FAR)], ids=str)
def test_append_output_on_other_operands(lib, change):
    call = {**APPEND, "q": FAR, "k": 2 * FAR, "v": 3 * FAR, "kp": 5 * FAR, "vp": 6 * FAR, **change}
    assert lib.cb2_paged_append(*call.values()) == SHAPE


@pytest.mark.parametrize("change,want", [
    (dict(w=None), NULL), (dict(kept=None), NULL), (dict(budget=0), SHAPE), (dict(budget=17), SHAPE), (dict(first=-1), SHAPE),
    (dict(first=5, last=4), SHAPE), (dict(max_k=40), SHAPE), (dict(R=65536), SHAPE), (dict(page=0), SHAPE), (dict(dtype=5), DTYPE),
    (dict(k=P + 2), ALIGN), (dict(w=P + 4), ALIGN), (dict(vs=2052), ALIGN),
], ids=str)
def test_evict_refusals(lib, change, want):
    assert lib.cb2_paged_evict(*{**EVICT, **change}.values()) == want


@pytest.mark.parametrize("budget", [(1 << 30) + 1, (1 << 31) - 1024, (1 << 31) - 1])
def test_evict_budget_bound(lib, budget):
    # a kernel's loop over the budget steps by its threads in 32 bits
    assert lib.cb2_paged_evict(*{**EVICT, "budget": budget, "new_pages": 1 << 27}.values()) == SHAPE


def test_no_tokens_is_no_launch(lib):
    assert lib.cb2_om_paged_fwd(*{**ATTEND, "n": 0, "q": None, "o": None, "scratch": None, "bytes": 0}.values()) == 0
    assert lib.cb2_paged_append(*{**APPEND, "n": 0, "q": None, "k": None, "v": None}.values()) == 0
    assert lib.cb2_om_paged_scratch_bytes(0, 2, 4, 2, 64, 1, 32, 0, 1) == 0
    assert "index" in lib.cb2_status_str(C.c_int(8)).decode()


def test_host_tensors_are_refused():
    from catopt_b200 import B200Error, ops

    pool = torch.zeros(2, 2, 16, 64)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(B200Error):
        ops.om_paged_fwd(torch.zeros(1, 4, 64), pool, pool, i, i[0], torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(B200Error):
        ops.paged_append(None, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), pool, pool, i, i[0], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(B200Error):
        ops.paged_evict(pool, pool, pool[..., 0], i, i[0], i, 4)


# --------------------------------------------------------------------------- the cache's bookkeeping
def make(**kw):
    from catopt_b200.paged import PagedCache

    return PagedCache(**{**dict(n_layers=1, n_pages=10, page_size=8, n_kv_heads=1, head_dim=8, device="cpu", track_weights=True), **kw})


def test_cache_hands_out_and_takes_back_pages():
    from catopt_b200 import B200Error

    c = make()
    a, b = c.open(), c.open()
    s = c.begin({a: 9, b: 0})
    assert s.table.tolist()[0][:2] == [0, 1] and s.table.tolist()[1] == [-1, -1]
    assert s.seq_lens.tolist() == [9, 0] and s.cu_q.tolist() == [0, 9, 9] and s.positions.tolist() == list(range(9))
    assert (s.n_tokens, s.max_q, s.max_k) == (9, 9, 9)
    s = c.begin({b: 8, a: 7})                        # a's last page still has room, b fills one
    assert c.free_pages == 7 and s.seq_lens.tolist() == [8, 16]
    assert s.positions.tolist() == list(range(8)) + list(range(9, 16)) and s.requests == (b, a)
    with pytest.raises(B200Error, match="pages"):
        c.begin({a: 8, b: 100})
    assert c.length(a) == 16 and c.length(b) == 8 and c.free_pages == 7          # nothing has changed
    used = set(s.table.flatten().tolist()) - {-1}
    assert len(used) == 3
    c.close(a)
    assert c.free_pages == 9
    with pytest.raises(B200Error, match="not open"):
        c.begin({a: 1})
    again = c.begin({c.open(): 72})
    assert not set(again.table.flatten().tolist()) & set(s.table[0].tolist()[:1])     # b's page stays b's
    assert c.free_pages == 0


def test_cache_refusals():
    from catopt_b200 import B200Error

    for bad in (dict(page_size=12), dict(page_size=4), dict(head_dim=132), dict(head_dim=12), dict(n_pages=0), dict(dtype=torch.float16)):
        with pytest.raises(B200Error):
            make(**bad)
    c = make()
    r = c.open()
    for call in (lambda: c.begin({}), lambda: c.begin({r: -1}), lambda: c.begin({99: 1}), lambda: c.evict([r, r], 4),
                 lambda: c.evict([r], 0), lambda: c.evict([r], 4, keep_first=3, keep_last=2), lambda: make(track_weights=False).evict([], 4)):
        with pytest.raises(B200Error):
            call()
    assert c.evict([r], 4) == []                     # not longer than the budget: nothing to do
    c.begin({r: 60})                                 # 8 of 10 pages
    with pytest.raises(B200Error, match="free"):
        c.evict([r], 20)                             # the kept keys need 3 fresh ones
    assert c.length(r) == 60 and c.free_pages == 2


def fake_evict(k, v, w, table, lens, to, budget, *, keep_first, keep_last, max_k):
    """paged_evict on the host."""
    import paged_reference as ref

    page, kept = k.shape[2], torch.full((len(lens), k.shape[1], budget), -1, dtype=torch.int32)
    for r, n in enumerate(lens.tolist()):
        ids = table[r, :(n + page - 1) // page].long()
        assert (ids >= 0).all() and not set(to[r].tolist()) & set(table.flatten().tolist())
        for h in range(k.shape[1]):
            j = torch.tensor(ref.keep(w[ids, h].reshape(-1), n, budget, keep_first, keep_last))
            kept[r, h, :len(j)] = j
            i = torch.arange(len(j))
            for t in (k, v, w):
                t[to[r].long()[i // page], h, i % page] = t[ids[j // page], h, j % page]
    return kept, lens.clamp(max=budget)


def test_cache_evicts_when_few_pages_are_free(monkeypatch):
    # one fresh page serves requests one after the other: the pages of one that is cut are there for the next
    from catopt_b200 import ops

    monkeypatch.setattr(ops, "paged_evict", fake_evict)
    c = make(n_layers=2)
    a, b, d = c.open(), c.open(), c.open()
    s = c.begin({a: 40, b: 24, d: 8})                # 9 of 10 pages
    g = torch.Generator().manual_seed(1)
    for t in (*c.k, *c.weights):
        t.copy_(torch.rand(t.shape, generator=g))
    before = [[c.k[i][s.table[r, :n // 8].long(), 0].reshape(-1, 8).clone() for r, n in ((0, 40), (1, 24))] for i in range(2)]
    kept = c.evict([a, b, d], 8, keep_first=1, keep_last=2)
    assert [c.length(r) for r in (a, b, d)] == [8, 8, 8] and c.free_pages == 7
    assert [tuple(x.shape) for x in kept] == [(2, 1, 8)] * 2                       # d was not longer
    s = c.begin({a: 0, b: 0, d: 0})
    assert len(set(s.table[:, 0].tolist())) == 3
    for i in range(2):
        for r in range(2):
            assert torch.equal(c.k[i][int(s.table[r, 0]), 0], before[i][r][kept[i][r, 0].long()])


def test_cache_keeps_its_pages_when_a_call_fails(monkeypatch):
    from catopt_b200 import B200Error, ops

    c = make(n_layers=2)
    a, b = c.open(), c.open()
    c.begin({a: 20, b: 24})
    calls = []

    def failing(*args, **kw):
        calls.append(0)
        if len(calls) == 2:                          # the second layer
            raise B200Error("no")
        return fake_evict(*args, **kw)

    def state():
        return list(c._free), {r: list(p) for r, p in c._pages.items()}, dict(c._length), dict(c._position)

    was = state()
    monkeypatch.setattr(ops, "paged_evict", failing)
    with pytest.raises(B200Error, match="no"):
        c.evict([a, b], 8)
    assert state() == was
    monkeypatch.setattr(c, "_to_device", lambda *rows: (_ for _ in ()).throw(RuntimeError("no memory")))
    with pytest.raises(RuntimeError, match="no memory"):
        c.evict([a, b], 8)
    with pytest.raises(RuntimeError, match="no memory"):
        c.begin({a: 20, b: 1})
    assert state() == was


def test_cache_refuses_a_batch_whose_pages_are_gone(monkeypatch):
    from catopt_b200 import B200Error, ops

    for name in ("paged_append", "om_paged_fwd"):
        monkeypatch.setattr(ops, name, lambda *a, **kw: "done")
    monkeypatch.setattr(ops, "paged_evict", fake_evict)
    c, other = make(), make()
    a, b, d = c.open(), c.open(), c.open()
    x = torch.zeros(1, 1, 8)

    def taken(batch, cache=c):
        return cache.append(0, batch, x, x, x), cache.attend(0, batch, x)

    first = c.begin({a: 20})
    both = c.begin({a: 1, b: 8})
    third = c.begin({d: 3})
    assert taken(first) == taken(both) == taken(third) == ("done", "done")          # later steps take no page away
    assert c.evict([a, b], 30) == [] and taken(both) == ("done", "done")            # nobody was cut
    c.evict([a], 8)
    for call in (lambda: c.append(0, first, x, x, x), lambda: c.attend(0, both, x)):
        with pytest.raises(B200Error, match=f"request {a}"):
            call()
    fourth = c.begin({b: 1, a: 1})
    c.close(d)
    assert taken(fourth) == ("done", "done")
    with pytest.raises(B200Error, match=f"request {d}"):
        taken(third)
    other.open()
    with pytest.raises(B200Error, match="another cache"):
        taken(fourth, other)


def test_host_calls_leave_what_is_not_in_order(lib):
    """The one-step form of a call declines whatever it does not know, without an exception: the wrapper then says why."""
    from catopt_b200 import ops

    t = torch.zeros(2, 2, 16, 64)
    i = torch.zeros(2, 2, dtype=torch.int32)
    assert ops._host("om_paged_fwd")() is NotImplemented
    assert ops._host("om_paged_fwd")({}, t[0], t, t, i, i[0], i[0], 1, None, None, True, None, None) is NotImplemented
    assert ops._host("om_paged_fwd")(*[None] * 13) is NotImplemented
    assert ops._host("paged_append")(*["x"] * 18) is NotImplemented
    assert ops._host("paged_evict")({}, t, t, t, i, i[0], i, 1, 0, 0, 1 << 80) is NotImplemented


def test_host_module_follows_torch_and_python(tmp_path, monkeypatch):
    from catopt_b200 import build

    calls = []

    def compile_(cmd):
        calls.append(cmd)
        build.HOST.touch()

    monkeypatch.setattr(build, "HOST", tmp_path / "_host.so")
    monkeypatch.setattr(build.subprocess, "check_call", compile_)
    for version, tag, want in ((torch.__version__, "cpython-312", 1), (torch.__version__, "cpython-312", 1), ("9.9", "cpython-312", 2),
                               ("9.9", "cpython-399", 3), ("9.9", "cpython-399", 3)):
        monkeypatch.setattr(torch, "__version__", version)
        monkeypatch.setattr(build.sys.implementation, "cache_tag", tag)
        build._build_host(False)
        assert len(calls) == want
    assert build.HOST.exists()


def test_host_module_that_does_not_load(lib, monkeypatch):
    import sys

    import catopt_b200
    from catopt_b200 import B200Error, ops

    class Refuses:
        @staticmethod
        def find_spec(name, path=None, target=None):
            if name == "catopt_b200._host":
                raise ImportError("undefined symbol")

    monkeypatch.delattr(catopt_b200, "_host", raising=False)
    monkeypatch.delitem(sys.modules, "catopt_b200._host", raising=False)
    monkeypatch.setattr(sys, "meta_path", [Refuses, *sys.meta_path])
    with pytest.raises(B200Error, match="catopt_b200.build"):
        ops._host.__wrapped__("paged_append")


# --------------------------------------------------------------------------- index tensors of any content
CSRC = Path(__file__).resolve().parent.parent / "catopt_b200" / "csrc"
INT_MIN, INT_MAX = -(1 << 31), (1 << 31) - 1


@pytest.fixture(scope="module")
def host_lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("clamp")
    (d / "clamp.cpp").write_text('#include "paged_clamp.cuh"\nextern "C" int clamp(int a, int b, int l, int n, int q, int k, int* out) {\n'
                                 "  cb2::PagedReq r;\n  const bool ok = cb2::paged_clamp(a, b, l, n, q, k, &r);\n"
                                 "  out[0] = r.t0, out[1] = r.n, out[2] = r.len;\n  return ok;\n}\n"
                                 'extern "C" int meet(long long at, long long n, long long token, long long heads, long long head, int d, int size,\n'
                                 "                    long long to, long long bytes) {\n"
                                 "  return cb2::paged_rows_meet((void*)at, n, token, heads, head, d, size, (void*)to, bytes);\n}\n")
    subprocess.check_call(["g++", "-O2", "-fwrapv", "-shared", "-fPIC", f"-I{CSRC}", str(d / "clamp.cpp"), "-o", str(d / "clamp.so")])
    return C.CDLL(str(d / "clamp.so"))


@pytest.fixture(scope="module")
def clamp(host_lib):
    """The kernels' clamp of a request, compiled for the host: ``f(c0, c1, len, n_tokens, max_q, max_k)``."""
    f = host_lib.clamp

    def call(*a):
        out = (C.c_int * 3)()
        ok = f(*map(C.c_int, a), out)
        return bool(ok), *out

    return call


def test_no_index_leads_out_of_bounds(clamp):
    values = [INT_MIN, INT_MIN + 1, INT_MIN + 5, INT_MIN + 9, -900, -1, 0, 1, 5, 7, 8, 9, 900, INT_MAX - 8, INT_MAX - 1, INT_MAX]
    for c0, c1 in itertools.product(values, values):
        for n_tokens, max_q in ((8, 8), (8, 3), (8, 0), (1, INT_MAX), (INT_MAX, INT_MAX)):
            ok, t0, n, _ = clamp(c0, c1, 0, n_tokens, max_q, 1)
            assert 0 <= t0 <= n_tokens and 0 <= n <= max_q and t0 + n <= n_tokens, (c0, c1, n_tokens, max_q, t0, n)
            good = 0 <= c0 <= c1 <= n_tokens and c1 - c0 <= max_q
            assert ok == good, (c0, c1, n_tokens, max_q)
            if good:
                assert (t0, n) == (c0, c1 - c0)
    for length in values:
        for max_k in (1, 8, 1 << 30):
            ok, _, _, got = clamp(0, 0, length, 8, 8, max_k)
            assert got == min(max(length, 0), max_k) and ok == (got == length)


def test_where_rows_meet(host_lib):
    """Rows [n, heads, d] with strides against a run of bytes: exact along the longer stride, the rows' whole extent
    along the other."""
    d, size = 8, 2
    for n, token, heads, head in ((1, 0, 1, 0), (3, 0, 1, 0), (3, 0, 2, 0), (2, 0, 3, 24), (3, 40, 2, 8), (3, 8, 2, 40), (4, 8, 1, 0), (1, 8, 3, 24), (2, 16, 4, 8)):
        outer, inner = ((n, token), (heads, head)) if n == 1 or heads == 1 or token >= head else ((heads, head), (n, token))
        row = ((inner[0] - 1) * inner[1] + d) * size
        used = {a for i in range(outer[0]) for a in range(i * outer[1] * size, i * outer[1] * size + row)}
        for to in range(-70, max(used) + 20):
            for count in (1, 16, 70):
                got = host_lib.meet(C.c_longlong(FAR), *(C.c_longlong(x) for x in (n, token, heads, head)), d, size, C.c_longlong(FAR + to),
                                    C.c_longlong(count))
                assert got == (not used.isdisjoint(range(to, to + count))), (n, token, heads, head, to, count)


# --------------------------------------------------------------------------- kernels launched while the one before runs
def waiting_kernels():
    """``(name, parameters, body)`` of every kernel that waits for the one before it inside itself."""
    for path in sorted(CSRC.glob("*.cu")):
        text = path.read_text()
        for m in re.finditer(r"__global__.*?(\w+)\(([^()]*(?:\([^()]*\)[^()]*)*)\)\s*\{\n(.*?)\n\}\n", text, re.S):
            if "after_previous()" in m[3]:
                yield m[1], m[2], m[3]


def test_kernels_that_wait_read_ordinarily():
    """What the kernel before writes while this one is resident is not constant for its lifetime: neither ``const
    __restrict__`` nor ``__ldg``, which may be moved before the wait.  (Index tensors of the batch, which no
    kernel of the chain writes, are read so.)"""
    found = {}
    for name, params, body in waiting_kernels():
        constant = [p.strip() for p in params.split(",") if "__restrict__" in p and "const" in p.split("*")[0]]
        loads = [x for x in re.findall(r"__ldg\((.*)", body) if not re.match(r"(reinterpret_cast<[^>]*>\()?(batch\.(lens|cu|table)|a\.to_table)\b", x)]
        found[name] = constant + loads
    assert len(found) >= 5 and not any(found.values()), {k: v for k, v in found.items() if v}
