"""Paged-cache operators on the GPU against plain 64-bit forms (paged_reference), whose error bounds count
the roundings a kernel makes.  Needs a B200: run with ``-m gpu``."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    from catopt_b200 import build

    build.build()
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)


def close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / tol).max().item():.3g} of the bound"


def run_attend(dev, new, lens, kv, group, d, page, dtype, causal=True, weights=False, seed=0, strided=False, scale=None, **cache_kw):
    from catopt_b200 import ops

    c = ref.make_cache(lens, kv, page, d, dtype, dev, seed, **cache_kw)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    n, hq = sum(new), kv * group
    wide = (1.5 * torch.randn(n, hq + 3, d + 8, generator=g, device=dev)).to(dtype)
    q = wide[:, 1:hq + 1, 8:] if strided else wide[:, 1:hq + 1, 8:].contiguous()
    w0 = torch.rand(c["k"].shape[:3], generator=g, device=dev) if weights else None
    w = None if w0 is None else w0.clone()
    cu = ref.offsets(new, dev)
    o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, max(new), max_k=max(max(lens), 1), causal=causal,
                         weights=w, scale=scale)
    ops.check_device_status(dev)
    want, tol, ww, wtol = ref.attend(q, c, new, lens, d ** -0.5 if scale is None else scale, causal)
    close(o, want, tol, "o")
    if weights:
        close(w, w0.double() + ww, wtol + 2 * ref.U32 * (w0 + ww), "weights")
    return c, q, o, w


RAGGED = [
    ([1], [1]), ([1, 1, 0, 1], [7, 130, 0, 513]), ([5, 1, 17], [5, 64, 400]), ([3, 0, 1, 2], [0, 0, 1, 1]),
    ([40, 1, 129], [170, 259, 129]), ([300], [1000]), ([2, 4, 1, 3], [2, 70, 500, 33]),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new,lens", RAGGED, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("kv,group,d,page", [(2, 4, 64, 16), (1, 3, 80, 8), (3, 1, 128, 32), (1, 16, 40, 256), (2, 8, 128, 64)])
def test_attention(dev, dtype, new, lens, kv, group, d, page):
    run_attend(dev, new, lens, kv, group, d, page, dtype, weights=True, seed=len(new) + d)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [8, 24, 56, 72, 120])
def test_attention_head_widths(dev, dtype, d):
    run_attend(dev, [1, 30, 200], [90, 30, 700], 2, 3, d, 16, dtype, weights=True)
    run_attend(dev, [1, 2, 1], [90, 300, 70], 2, 3, d, 8, dtype, weights=True)


@pytest.mark.parametrize("d,group", [(64, 4), (128, 1), (40, 8), (96, 7), (128, 16)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 3, 64]), ([2, 1], [300, 33]), ([1], [9000])], ids=["steps", "two", "long"])
def test_few_rows_keep_their_probabilities(dev, d, group, new, lens):
    # the product with V takes more of a probability than bf16 holds (two halves: 2^-16), and o is rounded once
    if max(new) * group > 16:
        new = [1] * len(new)
    c, q, o, _ = run_attend(dev, new, lens, 2, group, d, 16, BF, seed=d)
    want, tol, _, _ = ref.attend(q, c, new, lens, d ** -0.5, True)
    spread, _, _, _ = ref.attend(q, {**c, "v": c["v"].abs()}, new, lens, d ** -0.5, True)
    close(o, want, tol - spread * (ref.half_step(BF) - 2.0 ** -16), "o")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new", [1, 40], ids=["step", "chunk"])
def test_a_nan_that_is_seen_shows(dev, dtype, new):
    from catopt_b200 import ops

    lens, n = [500, 500], [new, new]
    c = ref.make_cache(lens, 1, 16, 64, dtype, dev, 13)
    c["k"][c["table"][1, 3].long(), 0, 5] = float("nan")          # slot 53 of the second request
    q = torch.randn(2 * new, 4, 64, device=dev).to(dtype)
    o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], ref.offsets(n, dev), new)
    assert o[:new].isfinite().all() and o[new:].isnan().all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new,group", [(1, 1), (1, 4), (2, 8), (40, 4)])
@pytest.mark.parametrize("length", [90, 500, 6000])
def test_an_infinite_value_that_is_seen_shows(dev, dtype, new, group, length):
    # every probability is above zero, so the sum is infinite where a value is, with its sign, and finite elsewhere
    from catopt_b200 import ops

    c = ref.make_cache([length], 2, 16, 64, dtype, dev, 14)
    g = torch.Generator(device=dev).manual_seed(15)
    for slot, col, x in ((0, 3, float("inf")), (37, 4, -float("inf")), (length - new, 5, float("inf")), (length - new - 1, 6, -float("inf"))):
        c["v"][c["table"][0, slot // 16].long(), :, slot % 16, col] = x
    q = torch.randn(new, 2 * group, 64, generator=g, device=dev).to(dtype)
    q[0, 0] = 0          # probabilities that are the same, and powers of two where the length is one
    o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], ref.offsets([new], dev), new, max_k=length)
    assert (o[..., [3, 5]] == float("inf")).all() and (o[..., [4, 6]] == -float("inf")).all()
    rest = [i for i in range(64) if i not in (3, 4, 5, 6)]
    assert o[..., rest].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new,lens", [([1, 1], [200, 130]), ([50, 20], [200, 130])], ids=["step", "chunk"])
def test_requests_that_share_pages(dev, dtype, new, lens):
    # the second request's first pages are the first one's: reading them twice is fine
    from catopt_b200 import ops

    c = ref.make_cache(lens, 2, 16, 64, dtype, dev, 14)
    c["table"][1, :4] = c["table"][0, :4]
    q = torch.randn(sum(new), 4, 64, device=dev).to(dtype)
    o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], ref.offsets(new, dev), max(new))
    want, tol, _, _ = ref.attend(q, c, new, lens, 0.125, True)
    close(o, want, tol, "o")


@pytest.mark.parametrize("rot,interleaved", [(64, False), (64, True), (40, False)])
def test_append_in_place(dev, rot, interleaved):
    from catopt_b200 import ops

    c = ref.make_cache([300], 2, 16, 64, BF, dev, 15, fill=0.0)
    q = torch.randn(300, 6, 64, device=dev).to(BF)
    k = torch.randn(300, 2, 64, device=dev).to(BF)
    ang = torch.rand(300, rot // 2, device=dev) * 6
    kw = dict(q_weight=torch.rand(64, device=dev).to(BF), cos=ang.cos(), sin=ang.sin(), interleaved=interleaved,
              positions=torch.arange(300, dtype=torch.int32, device=dev))
    cu = ref.offsets([300], dev)
    want = ops.paged_append(q, k, k, c["k"], c["v"], c["table"], c["lens"], cu, **kw)
    got = ops.paged_append(q, k, k, c["k"], c["v"], c["table"], c["lens"], cu, out=q, **kw)
    assert got is q and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("group", [1, 5])
def test_attention_all_keys_visible(dev, dtype, group):
    # queries against another sequence's states: more rows than keys, too
    run_attend(dev, [33, 1, 70, 9], [20, 300, 129, 0], 2, group, 64, 16, dtype, causal=False, weights=True)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_attention_strided_rows_and_spaced_pages(dev, dtype):
    run_attend(dev, [9, 1, 140], [60, 200, 333], 2, 4, 64, 16, dtype, strided=True, page_gap=64, weights=True, scale=0.3)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new,lens,kv,group", [([1], [20000], 1, 2), ([1] * 37, [(97 * i) % 700 + 1 for i in range(37)], 2, 4),
                                               ([2], [9001], 2, 7), ([64], [6000], 1, 4), ([1] * 300, [3 + i % 50 for i in range(300)], 1, 1),
                                               ([509, 1, 411, 314], [2048, 700, 1363, 679], 2, 4), ([1100], [6000], 2, 3)],
                         ids=["long", "many", "two", "chunk", "r300", "pieces", "long-pieces"])
def test_attention_work_cut_over_keys(dev, dtype, new, lens, kv, group):
    run_attend(dev, new, lens, kv, group, 128 if kv == 2 else 64, 16, dtype, weights=True, fill=float("inf"))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_chunk_beside_many_single_tokens(dev, dtype):
    # enough keys for both kernels of a mixed batch in fp32
    run_attend(dev, [40] + [1] * 30 + [5], [400 + 7 * i for i in range(32)], 8, 2, 64, 16, dtype, weights=True)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("group", [20, 72, 128])
def test_many_heads_on_one(dev, dtype, group):
    run_attend(dev, [1, 0, 7, 40], [300, 5, 200, 150], 1 if group > 20 else 2, group, 64, 16, dtype, weights=True)


@pytest.mark.parametrize("group", [3, 5, 7, 33, 60])
def test_weights_beside_a_key_of_infinities(dev, group):
    # a key that every row scores -inf gets nothing, as one that every row scores very low does
    from catopt_b200 import ops

    lens, new = [400], [100]
    c = ref.make_cache(lens, 2, 16, 64, BF, dev, 18)
    g = torch.Generator(device=dev).manual_seed(19)
    q = torch.randn(100, 2 * group, 64, generator=g, device=dev).to(BF)
    q[..., 0] = -1.0
    page, at = c["table"][0, 70 // 16].long(), 70 % 16
    got = []
    for x in (float("inf"), 1e5):
        c["k"][page, :, at, 0] = x
        w = torch.zeros(c["k"].shape[:3], device=dev)
        o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], ref.offsets(new, dev), 100, max_k=400, weights=w)
        assert o.isfinite().all() and (w[page, :, at] == 0).all()
        got.append((o, w))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_weights_when_the_bound_on_keys_is_far_off(dev):
    # scores of 2.3 million possible keys are not kept: the weights are computed from the keys again
    from catopt_b200 import ops

    lens, new = [700, 5], [1, 1]
    c = ref.make_cache(lens, 2, 256, 64, BF, dev, 8)
    wide = torch.full((2, 9000), -1, dtype=torch.int32, device=dev)
    wide[:, :c["table"].shape[1]] = c["table"]
    q = torch.randn(2, 8, 64, device=dev).to(BF)
    w = torch.zeros(c["k"].shape[:3], device=dev)
    o = ops.om_paged_fwd(q, c["k"], c["v"], wide, c["lens"], ref.offsets(new, dev), 1, weights=w)
    ops.check_device_status(dev)
    want, tol, ww, wtol = ref.attend(q, c, new, lens, 0.125, True)
    close(o, want, tol, "o")
    close(w, ww, wtol, "weights")


def test_fp32_weights_when_the_bound_on_keys_is_far_off(dev):
    # the same in fp32, where the scores' buffer is as large: few rows from the keys again
    from catopt_b200 import ops

    lens, new = [700, 5, 0], [1, 2, 0]
    c = ref.make_cache(lens, 2, 256, 64, F32, dev, 8)
    wide = torch.full((3, 9000), -1, dtype=torch.int32, device=dev)
    wide[:, :c["table"].shape[1]] = c["table"]
    q = torch.randn(3, 8, 64, device=dev)
    w = torch.zeros(c["k"].shape[:3], device=dev)
    o = ops.om_paged_fwd(q, c["k"], c["v"], wide, c["lens"], ref.offsets(new, dev), 2, weights=w)
    ops.check_device_status(dev)
    want, tol, ww, wtol = ref.attend(q, c, new, lens, 0.125, True)
    close(o, want, tol, "o")
    close(w, ww, wtol, "weights")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_chunks_of_many_requests(dev, dtype):
    # more requests than a CTA has threads: the search for a share, and the weights' loop over requests, take several rounds
    new = [(5 * i) % 23 if i % 7 else 0 for i in range(600)]
    lens = [n + (11 * i) % 40 if n else 0 for i, n in enumerate(new)]
    assert max(new) * 2 > 16
    run_attend(dev, new, lens, 1, 2, 32, 8, dtype, weights=True)


def test_append_of_many_requests(dev):
    # more requests than threads of a CTA
    from catopt_b200 import ops

    new = [i % 3 for i in range(700)]
    lens = [n + i % 20 if n else 0 for i, n in enumerate(new)]
    c = ref.make_cache(lens, 2, 8, 16, F32, dev, 23, fill=0.0)
    k, v = (torch.randn(sum(new), 2, 16, device=dev) for _ in range(2))
    want = [c["k"].clone(), c["v"].clone()]
    t = 0
    for r, n in enumerate(new):
        for j in range(lens[r] - n, lens[r]):
            p = int(c["table"][r, j // 8])
            want[0][p, :, j % 8], want[1][p, :, j % 8] = k[t], v[t]
            t += 1
    ops.paged_append(None, k, v, c["k"], c["v"], c["table"], c["lens"], ref.offsets(new, dev))
    ops.check_device_status(dev)
    assert torch.equal(c["k"], want[0]) and torch.equal(c["v"], want[1])


def test_large_scores_and_ties(dev):
    # a few keys dominate; the running maximum moves late, then by a lot
    from catopt_b200 import ops

    d, n = 64, 700
    c = ref.make_cache([n], 1, 16, d, F32, dev, 3)
    for pool in ("k", "v"):
        c[pool] = c[pool].to(BF)
    c["k"][c["table"][0, 600 // 16].long(), 0, 600 % 16] = 6.0
    q = torch.full((1, 2, d), 2.0, dtype=BF, device=dev)
    q[0, 1] = -2.0
    o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], ref.offsets([1], dev), 1, max_k=n, scale=1.0)
    want, tol, _, _ = ref.attend(q, c, [1], [n], 1.0, True)
    close(o, want, tol, "o")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_attention_same_bits_and_untouched_rows(dev, dtype):
    from catopt_b200 import ops

    new, lens = [1, 60, 1, 16], [900, 500, 40, 2000]
    c, q, o, _ = run_attend(dev, new, lens, 2, 4, 64, 16, dtype)
    cu = ref.offsets(new, dev)
    more = torch.cat([q, torch.full((5, *q.shape[1:]), float("nan"), dtype=dtype, device=dev)])
    out = torch.full_like(more, 7.0)
    again = ops.om_paged_fwd(more, c["k"], c["v"], c["table"], c["lens"], cu, 60, max_k=2000, out=out)
    assert again is out
    assert torch.equal(out[:q.shape[0]], o) and (out[q.shape[0]:] == 7.0).all()


def test_attention_graph_follows_lengths(dev):
    """A captured call reads lengths, offsets and table when it is replayed; two graphs share nothing."""
    from catopt_b200 import ops

    lens = [300, 90]
    c = ref.make_cache(lens, 2, 16, 64, BF, dev, 5)
    q = torch.randn(6, 8, 64, device=dev).to(BF)
    cu = ref.offsets([1, 5], dev)
    w = torch.zeros(c["k"].shape[:3], device=dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    with torch.cuda.stream(stream):
        for _ in range(2):
            ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 6, max_k=300, weights=w)
        for _ in range(2):
            gph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gph, stream=stream):
                outs.append(ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 6, max_k=300, weights=w))
            graphs.append(gph)
    torch.cuda.synchronize()
    for new, lens in (([1, 5], [300, 90]), ([4, 2], [77, 10]), ([6, 0], [250, 0])):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(ref.offsets(new, dev))
        w.zero_()
        for gph in graphs:
            gph.replay()
        torch.cuda.synchronize()
        ops.check_device_status(dev)
        want, tol, ww, wtol = ref.attend(q, c, new, lens, 0.125, True)
        for o in outs:
            close(o, want, tol, "o")
        close(w, 2 * ww, 2 * wtol + 4 * ref.U32 * ww, "weights")


def test_bad_indices_are_reported(dev):
    from catopt_b200 import B200Error, ops

    for dtype in (BF, F32):
        c = ref.make_cache([40, 70], 2, 16, 64, dtype, dev, 6, fill=0.0)
        q = torch.randn(3, 4, 64, device=dev).to(dtype)
        cu = ref.offsets([1, 2], dev)
        good = ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 2)
        ops.check_device_status(dev)

        def bad(table=None, lens=None, cu_q=None):
            o = ops.om_paged_fwd(q, c["k"], c["v"], c["table"] if table is None else table, c["lens"] if lens is None else lens,
                                 cu if cu_q is None else cu_q, 2)
            with pytest.raises(B200Error, match="index"):
                ops.check_device_status(dev)
            return o

        t = c["table"].clone()
        t[0, 0] = 1 << 30
        assert torch.equal(bad(table=t)[1:], good[1:])       # the other request is not touched by it
        t[0, 0] = -5
        bad(table=t)
        bad(lens=torch.tensor([40, 1 << 30], dtype=torch.int32, device=dev))
        bad(lens=torch.tensor([-3, 70], dtype=torch.int32, device=dev))
        bad(cu_q=torch.tensor([0, 1, 900], dtype=torch.int32, device=dev))
        bad(cu_q=torch.tensor([-7, 1, 3], dtype=torch.int32, device=dev))
        bad(cu_q=torch.tensor([0, 0, 3], dtype=torch.int32, device=dev))      # three new tokens where two were promised
        k = torch.randn(3, 2, 64, device=dev).to(dtype)
        t = c["table"].clone()
        t[1, 4] = c["k"].shape[0]
        before = c["k"].clone()
        ops.paged_append(None, k, k, c["k"], c["v"], t, c["lens"], cu)
        with pytest.raises(B200Error, match="index"):
            ops.check_device_status(dev)
        changed = (c["k"] != before).any(-1).any(1).sum().item()
        assert changed == 1                                    # request 0's token; request 1's have no page


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [8, 200], ids=["step", "chunk"])
def test_indices_of_any_content_stay_in_bounds(dev, dtype, n):
    # extremes of int32, whose differences do not fit it: reported, nothing behind the outputs is written
    from catopt_b200 import B200Error, ops

    lo, hi = -(1 << 31), (1 << 31) - 1
    c = ref.make_cache([300, 70], 1, 16, 64, dtype, dev, 16, fill=0.0)
    q = torch.randn(n, 2, 64, device=dev).to(dtype)
    k = torch.randn(n, 1, 64, device=dev).to(dtype)
    rest = [torch.full((n + 64, 2, 64), 5.0, dtype=dtype, device=dev) for _ in range(2)]
    w = torch.zeros(c["k"].shape[:3], device=dev)
    for cu in ([0, 5, lo], [0, lo, 5], [lo, 5, n], [0, hi, lo], [5, hi, n], [hi, lo, hi]):
        for lens in ([300, 70], [lo, hi]):
            cu_q, seq = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (cu, lens))
            ops.om_paged_fwd(q, c["k"], c["v"], c["table"], seq, cu_q, n, max_k=300, weights=w, out=rest[0][:n])
            with pytest.raises(B200Error, match="index"):
                ops.check_device_status(dev)
            ops.paged_append(q, k, k, c["k"], c["v"], c["table"], seq, cu_q, weights=w, out=rest[1][:n])
            torch.cuda.synchronize()
            ops.device_status(dev).zero_()
            assert all((x[n:] == 5.0).all() for x in rest)


# --------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new,start", [([1], [0]), ([3, 0, 1, 20], [5, 0, 16, 30]), ([700, 1, 2500], [0, 31, 8])],
                         ids=["one", "ragged", "many"])
@pytest.mark.parametrize("d,rot,interleaved,norm", [(128, 128, False, True), (80, 40, True, False), (64, 0, False, True),
                                                    (40, 20, False, True), (128, 96, True, True)])
@pytest.mark.parametrize("strided", [False, True], ids=["dense", "fused"])
def test_append(dev, dtype, new, start, d, rot, interleaved, norm, strided):
    from catopt_b200 import ops

    kv, hq, page = 2, 6, 16
    lens = [a + b if a else 0 for a, b in zip(new, start)]
    c = ref.make_cache(lens, kv, page, d, dtype, dev, 11, fill=3.0)
    g = torch.Generator(device=dev).manual_seed(d)
    n = sum(new)
    extra = 4                                    # rows behind the last sequence
    x = torch.randn(n + extra, hq + 2 * kv, d, generator=g, device=dev).to(dtype)
    q, k, v = x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qw = kw = cos = sin = pos = None
    if norm:
        qw, kw = (1 + 0.2 * torch.randn(d, generator=g, device=dev).to(dtype) for _ in range(2))
    if rot:
        ang = torch.rand(5000, rot // 2, generator=g, device=dev) * 6.3
        cos, sin = ang.cos(), ang.sin()
        pos = torch.randint(0, 5000, (n + extra,), generator=g, device=dev, dtype=torch.int32)
    w = torch.rand(c["k"].shape[:3], generator=g, device=dev)
    before = [t.clone() for t in (c["k"], c["v"], w)]
    out = torch.full((n + extra, hq, d), 9.0, dtype=dtype, device=dev)
    cu = ref.offsets(new, dev)
    got = ops.paged_append(q, k, v, c["k"], c["v"], c["table"], c["lens"], cu, q_weight=qw, k_weight=kw, eps=1e-5, cos=cos, sin=sin,
                           positions=pos, interleaved=interleaved, weights=w, out=out)
    ops.check_device_status(dev)
    wq, tq = ref.turned(q[:n], qw, 1e-5, cos, sin, None if pos is None else pos[:n], interleaved)
    wk, tk = ref.turned(k[:n], kw, 1e-5, cos, sin, None if pos is None else pos[:n], interleaved)
    assert got is out
    close(out[:n], wq, tq, "q")
    assert (out[n:] == 9.0).all()
    want_k, want_v, want_w = before
    tol_k = torch.zeros(want_k.shape, dtype=torch.float64, device=dev)
    want_k = want_k.double()
    t = 0
    for r, x in enumerate(new):
        for j in range(lens[r] - x, lens[r]):
            p, s = int(c["table"][r, j // page]), j % page
            want_k[p, :, s], tol_k[p, :, s], want_v[p, :, s] = wk[t], tk[t], v[t]
            want_w[p, :, s] = 0
            t += 1
    close(c["k"], want_k, tol_k, "k pages")
    assert torch.equal(c["v"], want_v) and torch.equal(w, want_w)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d,rot", [(64, 40), (40, 4), (128, 126)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("fill", [float("inf"), float("nan")], ids=["inf", "nan"])
def test_append_leaves_columns_behind_the_rotation(dev, dtype, d, rot, interleaved, fill):
    # columns that are not rotated come out as they went in, whatever stands beside them
    from catopt_b200 import ops

    c = ref.make_cache([9], 2, 16, d, dtype, dev, 17, fill=0.0)
    q, k = (torch.randn(9, h, d, device=dev).to(dtype) for h in (3, 2))
    for x in (q, k):
        x[..., rot::2] = fill
    ang = torch.rand(9, rot // 2, device=dev) * 6
    got = ops.paged_append(q, k, k, c["k"], c["v"], c["table"], c["lens"], ref.offsets([9], dev), cos=ang.cos(), sin=ang.sin(),
                           positions=torch.arange(9, dtype=torch.int32, device=dev), interleaved=interleaved)
    stored = c["k"][c["table"][0, 0].long(), :, :9].transpose(0, 1)
    for x, y in ((q, got), (k, stored)):
        assert torch.equal(x[..., rot:].nan_to_num(7.0), y[..., rot:].nan_to_num(7.0)) and y[..., :rot].isfinite().all()


@pytest.mark.parametrize("cu", [[0, 5, 3, 8], [0, 8, 2, 8], [3, 0, 8, 8], [0, 8, 9, 9], [0, 8, 8, -1]])
def test_append_reports_offsets_out_of_order(dev, cu):
    from catopt_b200 import B200Error, ops

    c = ref.make_cache([40, 70, 30], 2, 16, 64, F32, dev, 6, fill=0.0)
    k = torch.randn(8, 2, 64, device=dev)
    ops.paged_append(None, k, k, c["k"], c["v"], c["table"], c["lens"], torch.tensor(cu, dtype=torch.int32, device=dev))
    with pytest.raises(B200Error, match="index"):
        ops.check_device_status(dev)


# --------------------------------------------------------------------------- evict
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,budget,first,last", [
    ([5, 1, 40, 0], 8, 2, 3), ([300, 17, 16, 33], 16, 0, 0), ([700], 200, 4, 64), ([64, 65], 64, 32, 32), ([2500, 1300], 1111, 1, 0),
    ([9000], 4096, 16, 100), ([20], 1, 0, 1)])
@pytest.mark.parametrize("kv,d,page", [(2, 64, 16), (3, 40, 8), (1, 128, 128)])
def test_evict(dev, dtype, lens, budget, first, last, kv, d, page):
    from catopt_b200 import ops

    need = (budget + page - 1) // page
    c = ref.make_cache(lens, kv, page, d, dtype, dev, 21, fill=float("nan"), spare=need * len(lens) + 2)
    g = torch.Generator(device=dev).manual_seed(sum(lens))
    w = torch.randn(c["k"].shape[:3], generator=g, device=dev)
    w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.3, (w * 2).round() / 2, w)     # ties, and both zeros
    w[torch.rand(w.shape, generator=g, device=dev) < 0.02] = float("nan")
    w[torch.rand(w.shape, generator=g, device=dev) < 0.02] = float("inf")
    to = torch.tensor(c["free"][:need * len(lens)], dtype=torch.int32, device=dev).view(len(lens), need)
    want = [t.clone() for t in (c["k"], c["v"], w)]
    kept_want = torch.full((len(lens), kv, budget), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        for h in range(kv):
            ids = c["table"][r, :(n + page - 1) // page].long()
            kept = ref.keep(w[ids, h].reshape(-1).cpu(), n, budget, first, last)
            kept_want[r, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            j = torch.tensor(kept, device=dev, dtype=torch.long)
            i = torch.arange(len(kept), device=dev)
            for t in want:
                t[to[r].long()[i // page], h, i % page] = t[ids[j // page], h, j % page]
    kept, new_lens = ops.paged_evict(c["k"], c["v"], w, c["table"], c["lens"], to, budget, keep_first=first, keep_last=last)
    ops.check_device_status(dev)
    assert torch.equal(kept.cpu(), kept_want)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    bits = {2: torch.int16, 4: torch.int32}
    for got, exp in zip((c["k"], c["v"], w), want):
        assert torch.equal(got.view(bits[got.element_size()]), exp.view(bits[exp.element_size()]))


@pytest.mark.parametrize("budget", [1000, 49200, 52000])
def test_evict_from_more_keys_than_shared_memory_holds(dev, budget):
    # 49152 keys are held, the others read again in every pass; many ties, kept and dropped ones on both sides
    from catopt_b200 import ops

    n, d, page, first, last = 53000, 8, 64, 3, 40
    need = (budget + page - 1) // page
    c = ref.make_cache([n], 1, page, d, F32, dev, 31, fill=0.0, spare=need)
    g = torch.Generator(device=dev).manual_seed(budget)
    w = torch.randint(0, 50, c["k"].shape[:3], generator=g, device=dev).float() / 8
    to = torch.tensor([c["free"]], dtype=torch.int32, device=dev)
    ids = c["table"][0, :(n + page - 1) // page].long()
    want = ref.keep(w[ids, 0].reshape(-1).cpu(), n, budget, first, last)
    kept, new_lens = ops.paged_evict(c["k"], c["v"], w, c["table"], c["lens"], to, budget, keep_first=first, keep_last=last)
    ops.check_device_status(dev)
    assert kept[0, 0].tolist() == want and new_lens.tolist() == [budget]
    assert budget == 1000 or 49152 < want[-last - 1]          # (the 960 lowest of the heaviest keys lie in front)
    for pool in (c["k"], c["v"], w.unsqueeze(-1)):
        rows = pool[ids, 0].reshape(-1, pool.shape[-1])[torch.tensor(want, device=dev)]
        assert torch.equal(pool[to[0].long(), 0].reshape(-1, pool.shape[-1])[:budget], rows)


# --------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("steps", [[40], [1] * 12, [200, 1, 30, 1]], ids=["chunk", "tokens", "both"])
def test_eviction_by_the_weights_that_attention_leaves(dev, dtype, steps):
    """Against 64-bit sums over the keys that the cache holds: what is kept is not lighter than what is dropped, but by
    the error bounds of two sums."""
    from catopt_b200.paged import PagedCache

    kv, group, d, budget, first, last = 2, 3, 64, 24, 2, 4
    g = torch.Generator(device=dev).manual_seed(5)
    cache = PagedCache(1, 40, 16, kv, d, dtype=dtype, device=dev, track_weights=True)
    r, other = cache.open(), cache.open()
    total, bound = (torch.zeros(40, kv, 16, dtype=torch.float64, device=dev) for _ in range(2))
    for n in [30, *steps]:
        batch = cache.begin({other: 1, r: n})
        x = torch.randn(n + 1, kv * (group + 2), d, generator=g, device=dev).to(dtype)
        cache.append(0, batch, None, x[:, -2 * kv:-kv], x[:, -kv:])
        q = x[:, :kv * group]
        cache.attend(0, batch, q)
        held = {"k": cache.k[0], "v": cache.v[0], "table": batch.table, "page": 16}
        _, _, w, tol = ref.attend(q, held, [1, n], batch.seq_lens.tolist(), d ** -0.5, True)
        total += w
        bound += tol + 2 * ref.U32 * total          # one more addition
    length = cache.length(r)
    assert budget < length
    ids = batch.table[1, :(length + 15) // 16].long()
    sums, bounds = (t[ids].transpose(0, 1).reshape(kv, -1)[:, :length] for t in (total, bound))
    close(cache.weights[0][ids].transpose(0, 1).reshape(kv, -1)[:, :length], sums, bounds, "weights")
    kept = cache.evict([r], budget, keep_first=first, keep_last=last)[0][0].long()
    for h in range(kv):
        assert kept[h].tolist() == sorted(set(kept[h].tolist()))
        dropped = torch.ones(length, dtype=torch.bool, device=dev)
        dropped[kept[h]] = False
        assert not dropped[:first].any() and not dropped[length - last:].any()
        assert (sums + bounds)[h][kept[h, first:-last]].min() >= (sums - bounds)[h][dropped].max()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_decode_loop(dev, dtype):
    """Prompts in chunks, single tokens, an eviction, more tokens, a request that ends and one that begins: every output
    against 64-bit attention over lists of keys kept beside the cache."""
    from catopt_b200 import ops
    from catopt_b200.paged import PagedCache

    kv, group, d, layers = 2, 4, 64, 2
    hq = kv * group
    g = torch.Generator(device=dev).manual_seed(77)
    cache = PagedCache(layers, 64, 16, kv, d, dtype=dtype, device=dev, track_weights=True)
    ang = torch.arange(400, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2, device=dev, dtype=torch.float64) / (d // 2))
    cos, sin = ang.cos().float(), ang.sin().float()
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g, device=dev)).to(dtype) for _ in range(2))
    kept_keys = {}       # (request, layer, head) -> [keys], [values], [weights] in 64 bits

    def step(new):
        batch = cache.begin(new)
        n = sum(new.values())
        for layer in range(layers):
            x = torch.randn(n, hq + 2 * kv, d, generator=g, device=dev).to(dtype)
            q, k, v = x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:]
            qq = cache.append(layer, batch, q, k, v, q_weight=qw, k_weight=kw, cos=cos, sin=sin)
            o = cache.attend(layer, batch, qq)
            want_q, tol_q = ref.turned(q, qw, 1e-6, cos, sin, batch.positions, False)
            close(qq, want_q, tol_q, "q")
            want_k, _ = ref.turned(k, kw, 1e-6, cos, sin, batch.positions, False)
            want_k = want_k.to(dtype).double()          # what a cache of this type holds
            at = 0
            for r, m in new.items():
                for h in range(kv):
                    ks, vs, ws = kept_keys.setdefault((r, layer, h), ([], [], []))
                    ks += list(want_k[at:at + m, h])
                    vs += list(v[at:at + m, h].double())
                    ws += [0.0] * m
                    if not m:
                        continue
                    K, V = torch.stack(ks), torch.stack(vs)
                    s = torch.einsum("tgd,jd->gtj", qq[at:at + m, h * group:(h + 1) * group].double(), K) * d ** -0.5
                    t = len(ks) - m + torch.arange(m, device=dev)
                    s = s.masked_fill(torch.arange(len(ks), device=dev)[None, None] > t[None, :, None], float("-inf"))
                    p = torch.softmax(s, -1)
                    want = torch.einsum("gtj,jd->tgd", p, V)
                    spread = torch.einsum("gtj,jd->tgd", p, V.abs())
                    # a cached key may be one step of the type off its 64-bit rounding: 2 half steps of each score, 8 of
                    # which in magnitude are at most the sums below
                    dot = torch.einsum("tgd,jd->tgj", qq[at:at + m, h * group:(h + 1) * group].double().abs(), K.abs()).amax(-1, keepdim=True) * d ** -0.5
                    rel = 2 * dot * (2 * ref.half_step(dtype) + (d + 4) * ref.U32) + 2.0 ** -20
                    close(o[at:at + m, h * group:(h + 1) * group], want, spread * (rel + 2 * ref.half_step(dtype)) + 1e-6, "o")
                    ws[:] = (torch.tensor(ws, dtype=torch.float64, device=dev) + p.sum((0, 1))).tolist()
                at += m

    a, b = cache.open(), cache.open()
    step({a: 37, b: 90})
    step({b: 33, a: 1})
    for _ in range(3):
        step({a: 1, b: 1})
    kept = cache.evict([a, b], 48, keep_first=2, keep_last=8)
    assert cache.length(a) == 41 and cache.length(b) == 48 and cache.position(b) == 126
    for layer in range(layers):
        for h in range(kv):
            ks, vs, ws = kept_keys[b, layer, h]
            j = kept[layer][0, h].tolist()
            out = [i for i in range(len(ks)) if i not in j]
            assert j[:2] == [0, 1] and j[-8:] == list(range(118, 126)) and j == sorted(j) and len(set(j)) == 48
            # the lightest kept key is not lighter than the heaviest evicted one, up to the rounding of the sums
            assert min(ws[i] for i in j[2:-8]) >= max(ws[i] for i in out) * (1 - (2.0 ** -4 if dtype == BF else 2.0 ** -12))
            kept_keys[b, layer, h] = [ks[i] for i in j], [vs[i] for i in j], [ws[i] for i in j]
    step({a: 1, b: 1})
    step({b: 20, a: 3})
    cache.close(a)
    c = cache.open()
    step({c: 50, b: 1})
    step({c: 0, b: 2})
    ops.check_device_status(dev)


def test_calls_on_two_streams(dev):
    """Calls on different streams share nothing; tensors of another stream's making are ordered by the caller."""
    from catopt_b200 import ops

    c = ref.make_cache([1500, 700], 2, 16, 64, BF, dev, 9)
    cu = ref.offsets([1, 120], dev)
    qs = [torch.randn(121, 8, 64, device=dev).to(BF) for _ in range(2)]
    want = [ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 120) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.om_paged_fwd(qs[i], c["k"], c["v"], c["table"], c["lens"], cu, 120))
    torch.cuda.synchronize()
    ops.check_device_status(dev)
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_gradients_are_refused(dev):
    from catopt_b200 import B200Error, ops

    c = ref.make_cache([20], 1, 16, 64, BF, dev, 10)
    cu = ref.offsets([1], dev)
    q = torch.randn(1, 2, 64, device=dev).to(BF).requires_grad_()
    with pytest.raises(B200Error, match="no_grad"):
        ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 1)
    with torch.no_grad():
        ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 1)
    k = torch.randn(1, 1, 64, device=dev).to(BF)
    with pytest.raises(B200Error, match="no_grad"):
        ops.paged_append(q, k, k, c["k"], c["v"], c["table"], c["lens"], cu)


def test_tangents_are_refused(dev):
    import torch.autograd.forward_ad as fwd
    from catopt_b200 import B200Error, ops

    c = ref.make_cache([20], 1, 16, 64, F32, dev, 10)
    cu = ref.offsets([1], dev)
    q, k = torch.randn(1, 2, 64, device=dev), torch.randn(1, 1, 64, device=dev)
    with fwd.dual_level():
        dual = [fwd.make_dual(x, torch.ones_like(x)) for x in (q, k)]
        for call in (lambda: ops.om_paged_fwd(dual[0], c["k"], c["v"], c["table"], c["lens"], cu, 1),
                     lambda: ops.paged_append(q, dual[1], k, c["k"], c["v"], c["table"], c["lens"], cu),
                     lambda: ops.paged_append(dual[0].mT.contiguous().mT, k, k, c["k"], c["v"], c["table"], c["lens"], cu)):
            with pytest.raises(B200Error, match="no gradient"):
                call()
        ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 1)


def test_tables_that_ask_for_a_gradient_are_refused(dev):
    from catopt_b200 import B200Error, ops

    c = ref.make_cache([20], 1, 16, 64, F32, dev, 10)
    cu = ref.offsets([1], dev)
    k = torch.randn(1, 1, 64, device=dev)
    cos, sin = (torch.randn(4, 32, device=dev) for _ in range(2))
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    w = torch.zeros(c["k"].shape[:3], device=dev)
    q = torch.randn(1, 2, 64, device=dev)
    grad = lambda x: x.clone().requires_grad_()
    for call in (lambda: ops.paged_append(None, k, k, c["k"], c["v"], c["table"], c["lens"], cu, cos=grad(cos), sin=sin, positions=pos),
                 lambda: ops.paged_append(None, k, k, c["k"], c["v"], c["table"], c["lens"], cu, weights=grad(w)),
                 lambda: ops.paged_append(q, k, k, c["k"], c["v"], c["table"], c["lens"], cu, out=grad(q)),
                 lambda: ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 1, weights=grad(w)),
                 lambda: ops.om_paged_fwd(q, c["k"], c["v"], c["table"], c["lens"], cu, 1, out=grad(q))):
        with pytest.raises(B200Error, match="no gradient"):
            call()


def test_a_pool_of_one_page(dev):
    # the distance to a second page that is not there has no meaning
    from catopt_b200 import ops

    wide = torch.zeros(2 * 16 * 64 + 3, dtype=BF, device=dev)
    k, v = (wide.new_zeros(wide.shape).as_strided((1, 2, 16, 64), (x, 16 * 64, 64, 1)) for x in (2 * 16 * 64 + 3, 2 * 16 * 64 + 1))
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    lens = torch.tensor([10], dtype=torch.int32, device=dev)
    cu = ref.offsets([10], dev)
    x = torch.randn(10, 2, 64, device=dev).to(BF)
    w = torch.zeros(1, 2, 16, device=dev)
    ops.paged_append(None, x, x, k, v, table, lens, cu, weights=w)
    o = ops.om_paged_fwd(x, k, v, table, lens, cu, 10, weights=w)
    assert torch.equal(k[0, :, :10].transpose(0, 1), x) and torch.equal(o[0], x[0])


def test_wrong_arguments_are_refused(dev):
    from catopt_b200 import B200Error, ops

    c = ref.make_cache([20, 9], 2, 16, 64, BF, dev, 12)
    cu = ref.offsets([1, 1], dev)
    q = torch.randn(2, 4, 64, device=dev).to(BF)
    k = torch.randn(2, 2, 64, device=dev).to(BF)
    ok = dict(q=q, k_pages=c["k"], v_pages=c["v"], block_table=c["table"], seq_lens=c["lens"], cu_q=cu, max_q=1)
    ops.om_paged_fwd(**ok)
    for bad in (dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(v_pages=c["v"][:-1]), dict(k_pages=c["k"].transpose(1, 2)),
                dict(block_table=c["table"].long()), dict(seq_lens=c["lens"][:1]), dict(cu_q=cu[:2]), dict(max_k=1 << 20), dict(max_q=-1),
                dict(scale=-1.0), dict(weights=torch.zeros(3, device=dev)), dict(out=q), dict(out=torch.empty_like(q).float()), dict(seq_lens=c["lens"].cpu())):
        with pytest.raises(B200Error):
            ops.om_paged_fwd(**{**ok, **bad})
    ok = dict(q=q, k=k, v=k, k_pages=c["k"], v_pages=c["v"], block_table=c["table"], seq_lens=c["lens"], cu_q=cu)
    table = torch.zeros(8, 16, device=dev)
    for bad in (dict(k=k[:1]), dict(v=k.float()), dict(q=q[:1]), dict(cos=table), dict(cos=table, sin=table), dict(q_weight=torch.ones(64, device=dev)),
                dict(cos=table, sin=table, positions=torch.zeros(3, dtype=torch.int32, device=dev)), dict(eps=-1.0),
                dict(cos=table.repeat(1, 4), sin=table.repeat(1, 4), positions=cu[:2])):
        with pytest.raises(B200Error):
            ops.paged_append(**{**ok, **bad})
    w = torch.zeros(c["k"].shape[:3], device=dev)
    to = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    for bad in (dict(budget=17), dict(budget=0), dict(budget=8, keep_first=9), dict(budget=8, keep_first=4, keep_last=5), dict(budget=8, max_k=1 << 20)):
        with pytest.raises(B200Error):
            ops.paged_evict(c["k"], c["v"], w, c["table"], c["lens"], to, **bad)
    ops.check_device_status(dev)


def test_one_step_calls_and_the_wrappers_agree(dev, monkeypatch):
    """A call in order is checked and launched in one step (host_calls.cpp); the wrapper's own rules, when they are
    gone through, give the same answer.  What needs the wrapper is left to it."""
    from catopt_b200 import ops

    ops.device_status(dev)
    lens, new = [70, 33], [5, 1]
    c = ref.make_cache(lens, 2, 16, 64, BF, dev, 3, fill=0.0)
    cu = ref.offsets(new, dev)
    g = torch.Generator(device=dev).manual_seed(4)
    q, k, v = (torch.randn(6, h, 64, generator=g, device=dev).to(BF) for h in (4, 2, 2))
    cos, sin = (torch.randn(80, 16, generator=g, device=dev) for _ in range(2))
    pos = torch.arange(6, dtype=torch.int32, device=dev)
    qw, kw = (torch.randn(64, generator=g, device=dev).to(BF) for _ in range(2))
    weights = torch.rand(c["k"].shape[:3], generator=g, device=dev)
    free = [p for p in range(c["k"].shape[0]) if p not in set(c["table"].flatten().tolist())][:2]
    assert len(free) == 2
    to = torch.tensor([[p] for p in free], dtype=torch.int32, device=dev)

    def run(**kw_attend):
        kp, vp, w = c["k"].clone(), c["v"].clone(), weights.clone()
        turned = ops.paged_append(q, k, v, kp, vp, c["table"], c["lens"], cu, q_weight=qw, k_weight=kw, cos=cos, sin=sin, positions=pos,
                                  weights=w)
        none = ops.paged_append(None, k, v, kp, vp, c["table"], c["lens"], cu)
        out = torch.empty_like(q)
        o = ops.om_paged_fwd(turned, kp, vp, c["table"], c["lens"], cu, 5, weights=w, out=out, **kw_attend)
        o2 = ops.om_paged_fwd(turned, kp, vp, c["table"], c["lens"], cu, 5, max_k=70, scale=0.25, causal=False)
        kept, lens2 = ops.paged_evict(kp, vp, w, c["table"], c["lens"], to, 16, keep_first=2, keep_last=4)
        assert none is None and o is out
        ops.check_device_status(dev)
        return [turned, o, o2, kept, lens2, kp, vp, w]

    taken = []
    with monkeypatch.context() as m:
        host = ops._host
        m.setattr(ops, "_host", lambda name: lambda *a: taken.append(host(name)(*a)) or taken[-1])
        one = run()
    assert len(taken) == 5 and not any(x is NotImplemented for x in taken)
    with monkeypatch.context() as m:
        m.setattr(ops, "_host", lambda name: lambda *a: NotImplemented)
        other = run()
    for a, b in zip(one, other):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    # not in order as they stand: rows to copy first, numbers of other kinds, gradients, shapes
    attend = (c["k"], c["v"], c["table"], c["lens"], cu)
    f = host("om_paged_fwd")
    assert f(ops._status_words, q.mT.contiguous().mT, *attend, 5, None, None, True, None, None) is NotImplemented
    assert f(ops._status_words, q, *attend, True, None, None, True, None, None) is NotImplemented
    assert f(ops._status_words, q, *attend, 5, None, 1, True, None, None) is NotImplemented
    assert f(ops._status_words, q, *attend, 5, 81 * 16, None, True, None, None) is NotImplemented
    assert f(ops._status_words, q, *attend, 5, None, None, True, weights[1:], None) is NotImplemented
    assert f({}, q, *attend, 5, None, None, True, None, None) is NotImplemented
    assert f(ops._status_words, q.clone().requires_grad_(), *attend, 5, None, None, True, None, None) is NotImplemented
    assert f(ops._status_words, q[:, :3], *attend, 5, None, None, True, None, None) is NotImplemented
    with pytest.raises(ops.B200Error):
        ops.om_paged_fwd(q, *attend, 5, out=q)           # declined by the entry point
    with pytest.raises(ops.B200Error):
        ops.om_paged_fwd(q, *attend, 5, scale=float("nan"))
