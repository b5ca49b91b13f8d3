"""Attention calls as a longer-lived program makes them: graphs kept over a shutdown, other streams, error words,
buffers in odd states.  (Results against the definitions: test_gpu_attn.py, whose helpers are used here.)"""

import threading
import time

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import ColizigError, attn, gpu, moe, synth  # noqa: E402
from tests.test_gpu_attn import Paged, close, gen, prefill_want, prompts, randn, softmax_rows  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def reported():
    """The error word as a check reports it: its code, or 0."""
    try:
        attn.check()
    except ColizigError as e:
        return e.rc
    return 0


def test_graph_kept_over_a_shutdown_reports_to_the_new_library():
    """A captured call holds the error word's address: it stays good after a shutdown and another init."""
    g = gen(70)
    pg = Paged(g, [100, 40], 2, 64, 16)
    q = randn(g, 2, 4, 64, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 4, 2)
    lens = pg.len_t.clone()
    want = plan.run(q, pg.table, lens)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.run(q, pg.table, lens, out=out)
    gpu.deinit()
    gpu.init()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and reported() == 0
    lens[1] = -1
    graph.replay()
    torch.cuda.synchronize()
    assert reported() == -11 and reported() == 0


def test_errors_after_a_check_s_read_are_kept_for_the_next():
    """A check queued behind a long kernel, a graph that meets a bad length queued behind the check's read while the
    check still waits: the first check reports what was there, the second the graph's."""
    g = gen(71)
    pg = Paged(g, [100, 40], 2, 64, 16)
    q = randn(g, 2, 4, 64, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 4, 2)
    bad = pg.len_t.clone()
    bad[0] = -5
    plan.run(q, pg.table, bad)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.run(q, pg.table, bad, out=out)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    first = []

    def check():
        try:
            attn.check(stream=s)
            first.append(0)
        except ColizigError as e:
            first.append(e.rc)

    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000_000)  # about a second
    t = threading.Thread(target=check)
    t.start()
    time.sleep(0.3)
    with torch.cuda.stream(s):
        graph.replay()
    t.join()
    s.synchronize()
    assert first == [-11]
    assert reported() == -11 and reported() == 0


def long_one(g, n=20000, hq=16, hk=2, d=128):
    """A sequence cut between blocks, its queries and the right answer."""
    pg = Paged(g, [n], hk, d, 64)
    q = randn(g, 1, hq, d, dtype=torch.bfloat16)
    want = attn.DecodePlan(pg.cache, hq, 1).run(q, pg.table, pg.len_t)
    torch.cuda.synchronize()
    return pg, q, want


def test_a_new_plan_runs_on_another_stream_at_once():
    """The workspace's zeros are queued on the stream where the plan is made, here behind a long kernel and over
    memory that held something else: a first call on another stream must find them."""
    pg, q, want = long_one(gen(72))
    size = attn.DecodePlan(pg.cache, 16, 1)._ws.numel()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    dirty = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    del dirty  # the plan's workspace takes its place
    torch.cuda._sleep(400_000_000)
    plan = attn.DecodePlan(pg.cache, 16, 1)
    got = plan.run(q, pg.table, pg.len_t, out=out, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    assert torch.equal(plan.run(q, pg.table, pg.len_t), want)


def test_a_plan_dropped_while_its_call_waits_on_another_current_stream():
    """The workspace is the plan's own: its memory is not handed out before the call on a stream that was made current
    has run."""
    pg, q, want = long_one(gen(73))
    plan = attn.DecodePlan(pg.cache, 16, 1)
    out = torch.zeros_like(want)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(400_000_000)
        plan.run(q, pg.table, pg.len_t, out=out)
    size = plan._ws.numel()
    del plan
    other = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del other


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("nq", [[4, 0, 300], [1], [30] * 40])
def test_prompts_on_no_keys_at_all(hq, hk, d, nq):
    """Zeros for every query of a sequence; rows past the last sequence's are not written, bad bounds are reported."""
    n = sum(nq)
    q = randn(gen(74), n + 5, hq, d, dtype=torch.bfloat16)
    kv = torch.empty((0, hk, d), device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0] + nq).cumsum(0).int().cuda()
    none = torch.zeros_like(cu)
    out = torch.full_like(q, 7.0)
    attn.prefill(q, kv, kv, cu, none, out=out)
    assert not out[:n].any() and (out[n:] == 7).all()
    assert reported() == 0
    for bad in ((cu, none.clone().index_fill_(0, torch.tensor([len(nq)], device="cuda"), 3)),
                (cu.clone().index_fill_(0, torch.tensor([len(nq)], device="cuda"), n + 6), none)):
        attn.prefill(q, kv, kv, *bad, out=out)
        assert reported() == -11
    assert (out[n:] == 7).all()


def test_decode_after_kernels_that_fill_shared_memory():
    """A block's flags start cleared whatever the kernel before left in shared memory (here rotated keys and products of
    all bits): no wait gives up early, results repeat."""
    g = gen(75)
    pg, q, want = long_one(g)
    plan = attn.DecodePlan(pg.cache, 16, 1)
    x, k, v, cu = prompts(g, [3000], [3000], 8, 2, 128, False)
    for _ in range(100):
        attn.prefill(x, k, v, cu[0])
        assert torch.equal(plan.run(q, pg.table, pg.len_t), want)
    assert reported() == 0


def test_calls_read_what_the_kernel_just_before_them_wrote():
    """The MoE decode kernel lets the kernel after it come before it has written anything. Its experts' numbers serve as
    decode's lengths and its output as the cache write's projections, both right behind it in a replayed graph."""
    gpu.init()
    g = gen(76)
    d = synth.CONFIGS["c1"]
    layer = moe.Layer.from_weights(830, d, synth.make_layer(d, seed=9, device="cuda"))
    try:
        x = synth.make_tokens(3, d.hidden, 1, device="cuda")
        out, idx = torch.empty((3, d.hidden), device="cuda"), torch.zeros((3, d.topk), dtype=torch.int32, device="cuda")
        gates = torch.empty((3, d.topk), device="cuda")
        lens = idx.view(-1)
        pg = Paged(g, [15] * lens.numel(), 2, 64, 16)
        q = randn(g, lens.numel(), 6, 64, dtype=torch.bfloat16)
        plan = attn.DecodePlan(pg.cache, 6, lens.numel())
        o = plan.run(q, pg.table, lens)
        cache = attn.KvCache.empty(1, 1, 16, 64)
        heads = out.view(3, 4, 64)
        slots = torch.arange(3, device="cuda")
        qo = attn.append(cache, heads[:, :2], heads[:, 2:3], heads[:, 3:], None, slots)[0]

        def both(first):
            moe.forward(layer, x, out, idx, gates)
            if first:
                plan.run(q, pg.table, lens, out=o)
            else:
                attn.append(cache, heads[:, :2], heads[:, 2:3], heads[:, 3:], None, slots, q_out=qo)

        graphs = []
        for first in (True, False):
            both(first)
            torch.cuda.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                both(first)
        seen = set()
        for i in range(20):
            x.copy_(synth.make_tokens(3, d.hidden, 100 + i, device="cuda"))
            graphs[0].replay()
            torch.cuda.synchronize()
            n = lens.tolist()
            seen.update(n)
            cut = Paged.__new__(Paged)
            cut.lens, cut.hk, cut.rows = n, pg.hk, [r[:, :k] for r, k in zip(pg.rows, n)]
            close(o, *cut.want(q, 64 ** -0.5))
            graphs[1].replay()
            torch.cuda.synchronize()
            assert torch.equal(qo, heads[:, :2].bfloat16())
            assert torch.equal(cache.k[0, 0, :3], heads[:, 2].bfloat16())
            assert torch.equal(cache.v[0, 0, :3], heads[:, 3].bfloat16())
        assert len(seen) > 8
        moe.check()
        assert reported() == 0
        del graphs
    finally:
        layer.unregister()


def one_key_each(g, n, d):
    """n keys of random signs: a key as a query has d as its product with itself and at most d - 2 with the others."""
    signs = torch.randint(0, 2, (n, d), generator=g, device="cuda") * 2 - 1
    return signs.to(torch.bfloat16)


@pytest.mark.parametrize("big", [2.0 ** 8, 2.0 ** 15, 2.0 ** 30, 2.0 ** 55])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_scores_of_any_size(big, d):
    """Scores far beyond those of trained weights, over several key tiles and rescalings: softmax leaves each query its
    one best key. (Signs times powers of two: the products are exact, two scores differ by 2 big^2 scale or not at
    all.)"""
    g = gen(77)
    n, hk, group = 700, 2, 4
    k = one_key_each(g, n * hk, d).view(n, hk, d)
    pick = (torch.rand((n, hk, group), generator=g, device="cuda") * (torch.arange(n, device="cuda")[:, None, None] + 1)).long()
    q = torch.stack([k[pick[:, h], h] for h in range(hk)], 1).reshape(n, hk * group, d)
    v = randn(g, n, hk, d, dtype=torch.bfloat16)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q, k = q * big, k * big
    got = attn.prefill(q, k, v, cu)
    close(got, *prefill_want(q, k, v, [n], [n], d ** -0.5))


@pytest.mark.parametrize("big", [2.0 ** 8, 2.0 ** 30, 2.0 ** 55])
def test_decode_scores_of_any_size(big):
    g = gen(78)
    pg = Paged(g, [900, 33], 2, 128, 64)
    for b, rows in enumerate(pg.rows):
        n = rows.shape[1]
        k = one_key_each(g, n * 2, 128).view(n, 2, 128) * big
        rows[0] = k.double()
        for i in range(-(-n // 64)):
            m = min(64, n - 64 * i)
            pg.cache.k[int(pg.table[b, i]), :, :m] = k[64 * i: 64 * i + m].transpose(0, 1)
    q = torch.stack([pg.rows[b][0][at].repeat_interleave(4, 0) for b, at in enumerate((611, 32))]).to(torch.bfloat16)
    got = attn.DecodePlan(pg.cache, 8, 2).run(q, pg.table, pg.len_t)
    close(got, *pg.want(q, 128 ** -0.5))


def test_two_plans_at_once_on_two_streams():
    a, b = long_one(gen(80)), long_one(gen(81), n=9001, hq=12, hk=4, d=64)
    plans = [attn.DecodePlan(pg.cache, q.shape[1], 1) for pg, q, _ in (a, b)]
    streams = [torch.cuda.Stream() for _ in plans]
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        for (pg, q, _), plan, s in zip((a, b), plans, streams):
            got.append(plan.run(q, pg.table, pg.len_t, stream=s))
    torch.cuda.synchronize()
    assert all(torch.equal(o, (a, b)[i % 2][2]) for i, o in enumerate(got))
    assert reported() == 0


def test_two_threads_with_a_plan_and_a_stream_each():
    ones = [long_one(gen(82)), long_one(gen(83), n=9001, hq=12, hk=4, d=64)]
    x, k, v, cu = prompts(gen(84), [500, 33], [500, 33], 8, 2, 64, False)
    whole = attn.prefill(x, k, v, cu[0])
    torch.cuda.synchronize()
    good = [0, 0]

    def work(i):
        pg, q, want = ones[i]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            plan = attn.DecodePlan(pg.cache, q.shape[1], 1)
            outs = [(plan.run(q, pg.table, pg.len_t), attn.prefill(x, k, v, cu[0])) for _ in range(60)]
            s.synchronize()
            good[i] = sum(torch.equal(o, want) and torch.equal(p, whole) for o, p in outs)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert good == [60, 60] and reported() == 0


@pytest.mark.parametrize("nq,nk", [([64], [8192]), ([1], [5000]), ([17, 200], [4097, 300])])
def test_prefill_of_a_short_chunk_on_many_keys(nq, nk):
    q, k, v, cu = prompts(gen(85), nq, nk, 32, 4, 128, False)
    got = attn.prefill(q, k, v, *cu)
    close(got, *prefill_want(q, k, v, nq, nk, 128 ** -0.5))


def test_a_prompt_in_chunks_through_the_cache():
    """Each chunk's keys are appended, all of them so far read back out of the pages and attended to."""
    g = gen(86)
    n, hq, hk, d, page = 333, 8, 2, 64, 16
    q, k, v, _ = prompts(g, [n], [n], hq, hk, d, False)
    cache = attn.KvCache.empty(-(-n // page), hk, page, d)
    order = torch.randperm(cache.pages, generator=torch.Generator().manual_seed(1)).cuda()
    at = 0
    for m in (100, 1, 200, 32):
        i = torch.arange(at, at + m, device="cuda")
        qo = attn.append(cache, q[i], k[i], v[i], None, order[i // page] * page + i % page)[0]
        at += m
        rows = [t[order].transpose(1, 2).reshape(-1, hk, d)[:at] for t in (cache.k, cache.v)]
        ends = [torch.tensor([0, e], dtype=torch.int32, device="cuda") for e in (m, at)]
        got = attn.prefill(qo, *rows, *ends)
        close(got, *prefill_want(q[at - m: at], k[:at], v[:at], [m], [at], d ** -0.5))


def test_decode_of_a_full_batch_on_e4m3():
    g = gen(87)
    lens = [1800 + 37 * i % 251 for i in range(64)]
    pg = Paged(g, lens, 4, 128, 64, True)
    q = randn(g, 64, 32, 128, dtype=torch.bfloat16) * 2
    got = attn.DecodePlan(pg.cache, 32, 64).run(q, pg.table, pg.len_t)
    close(got, *pg.want(q, 128 ** -0.5))


def test_scores_of_minus_infinity_leave_their_keys_out():
    """Keys of the type's lowest value, whose products with large queries are -infinity: as if they were masked; a row
    of nothing else gives zeros."""
    g = gen(88)
    n, d = 300, 128
    low = torch.finfo(torch.bfloat16).min
    q = torch.full((1, 8, d), 4.0, device="cuda", dtype=torch.bfloat16)
    k = randn(g, n, 1, d, dtype=torch.bfloat16)
    v = randn(g, n, 1, d, dtype=torch.bfloat16)
    out = torch.rand(n, generator=g, device="cuda") < 0.5
    k[out] = low
    o, w = softmax_rows(q[0], k[~out, 0], v[~out, 0], d ** -0.5, torch.ones(8, int((~out).sum()), dtype=torch.bool, device="cuda"))
    cache = attn.KvCache.empty(-(-n // 16), 1, 16, d)
    table = torch.arange(cache.pages, dtype=torch.int32, device="cuda")[None]
    one, all_n = (torch.tensor([0, e], dtype=torch.int32, device="cuda") for e in (1, n))
    for alone in (False, True):
        if alone:
            k[:] = low
        attn.append(cache, k.expand(n, 1, d), k, v, None, torch.arange(n, device="cuda"))
        got = [attn.DecodePlan(cache, 8, 1).run(q, table, all_n[1:]), attn.prefill(q, k, v, one, all_n)]
        for x in got:
            if alone:
                assert not x.any()
            else:
                close(x[0], o, w)


def microseconds(f, n=20):
    """Device time of a call in a replayed graph."""
    f()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for _ in range(n):
            f()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / n)
    return sorted(times)[3]


@pytest.mark.parametrize("nq,nk,hq,hk,d", [(700, 4700, 32, 4, 128), (1000, 4000, 32, 4, 128), (2500, 5000, 12, 2, 128)])
def test_a_chunk_takes_no_second_round_of_long_tiles(nq, nk, hq, hk, d):
    """Queries after many keys, whose tiles all are long: where pairs of tiles fill the SMs once, the call takes about as
    long as a pair alone on as many keys (an eighth of the queries), not twice that."""
    g = gen(89)

    def call(n):
        q, k, v, cu = prompts(g, [n], [nk], hq, hk, d, False)
        out = torch.empty_like(q)
        return lambda: attn.prefill(q, k, v, *cu, out=out)

    assert microseconds(call(nq)) < 1.6 * microseconds(call(nq // 8))
