"""The attention operators (colizig_b200.attn) against their definitions in 64 bits.

Tolerances, element by element, from how the results are made (bf16 holds 8 significant bits,
so a rounding is off by up to 2^-8 of the value).  Attention: the output is rounded to bf16
once (2^-8 of it) and each softmax weight may be rounded to bf16 before it multiplies its
value (2^-8 of sum p|v|); f32 scores of at most a few hundred are off by under
2^-12, which moves a weight by under 2^-12 of itself, and sums in f32 add less than that
again: 2^-11 of sum p|v| covers both.  append: f32 arithmetic of a dozen roundings (2^-20 of
the rotated pair's length) and one rounding to bf16 (2^-8) or E4M3 (2^-4 of the value, 2^-10
where E4M3 is subnormal; both times the head's scale)."""

import math

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import ColizigError, attn, gpu  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
NAN = float("nan")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def close(got, want, weight):
    """weight = sum p|v| (see above)."""
    got, want = got.double(), want.double()
    tol = want.abs() * 2.0 ** -8 + weight * (2.0 ** -8 + 2.0 ** -11)
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol).max()):.3e}"


def softmax_rows(q, k, v, scale, seen):
    """(o, sum p|v|) in f64 of q [r, d], k, v [n, d], seen [r, n]; zeros for rows that see nothing."""
    s = (q.double() @ k.double().T) * scale
    s = s.masked_fill(~seen, -math.inf)
    some = seen.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s))
    return p @ v.double(), p @ v.double().abs()


# ------------------------------------------------------------------ decode


class Paged:
    """A cache whose sequences lie on shuffled pages; whatever no sequence holds is NaN."""

    def __init__(self, g, lens, hk, d, page, e4m3=False, together=False, spare=3):
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        self.lens, self.page, self.hk, self.d = lens, page, hk, d
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(len(lens) + pages))
        self.width = max(1, max(need))
        table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = order[at:at + m].int()
            at += m
        self.table = table.cuda()
        kv = torch.full((2, pages, hk, page, d), NAN, device="cuda", dtype=torch.bfloat16)
        if together:  # keys and values of a page side by side in one allocation
            kv = torch.full((pages, 2, hk, page, d), NAN, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
        self.ks = self.vs = None
        if e4m3:
            self.ks = 0.01 + 0.02 * torch.rand(hk, generator=g, device="cuda")
            self.vs = 0.01 + 0.02 * torch.rand(hk, generator=g, device="cuda")
        self.rows = []
        for b, n in enumerate(lens):
            x = randn(g, 2, n, hk, d, dtype=torch.bfloat16)
            if e4m3:
                x = (x * 60).to(E4M3).to(torch.bfloat16)  # codes, exact in bf16
            for i in range(need[b]):
                m = min(page, n - i * page)
                kv[:, int(table[b, i]), :, :m] = x[:, i * page:i * page + m].transpose(1, 2)
            x = x.double()
            if e4m3:
                x = x * torch.stack([self.ks, self.vs]).double()[:, None, :, None]
            self.rows.append(x)
        if e4m3:
            kv = kv.to(E4M3)
        self.cache = attn.KvCache(kv[0], kv[1], self.ks, self.vs)
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def want(self, q, scale):
        hq = q.shape[1]
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        w = torch.zeros_like(o)
        for b, n in enumerate(self.lens):
            for h in range(hq):
                kh = h // (hq // self.hk)
                seen = torch.ones(1, n, dtype=torch.bool, device="cuda")
                if n:
                    r = softmax_rows(q[b, h][None], self.rows[b][0][:, kh], self.rows[b][1][:, kh], scale, seen)
                    o[b, h], w[b, h] = r[0][0], r[1][0]
        return o, w


LENS = [1, 0, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 1025]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 128), (32, 4, 128), (3, 3, 64), (10, 2, 128), (14, 2, 64), (24, 2, 128),
                                     (16, 1, 64), (20, 1, 128), (40, 1, 64), (33, 1, 128)])
def test_decode_head_layouts(hq, hk, d, e4m3):
    g = gen(hq * 7 + hk + d + e4m3)
    pg = Paged(g, LENS, hk, d, 16 if d == 64 else 64, e4m3)
    q = randn(g, len(LENS), hq, d, dtype=torch.bfloat16) * 2
    plan = attn.DecodePlan(pg.cache, hq, 64)
    got = plan.run(q, pg.table, pg.len_t)
    o, w = pg.want(q, d ** -0.5)
    close(got, o, w)
    assert not got[1].any()  # the empty sequence
    attn.check()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256, 1024])
def test_decode_page_sizes_and_strides(page, e4m3):
    g = gen(page + e4m3)
    lens = [page - 1, page, page + 1, 1, 2 * page + 7, 777, 0]
    pg = Paged(g, lens, 2, 128, page, e4m3, together=True)
    hq = 12
    # q as a slice of a wider row, the table as a slice of a wider table
    wide = randn(g, len(lens), hq + 5, 128, dtype=torch.bfloat16)
    q = wide[:, 2:2 + hq]
    table = torch.full((len(lens), pg.width + 3), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, :pg.width] = pg.table
    plan = attn.DecodePlan(pg.cache, hq, len(lens), scale=0.3)
    out = torch.full((len(lens), hq, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    got = plan.run(q, table, pg.len_t, out=out)
    assert got is out
    o, w = pg.want(q, 0.3)
    close(got, o, w)
    attn.check()


@pytest.mark.parametrize("lens", [[70001], [40000, 3], [9000] * 5 + [1] * 20, [513] * 300])
def test_decode_long_and_many(lens):
    g = gen(len(lens))
    pg = Paged(g, lens, 2, 64, 64)
    q = randn(g, len(lens), 16, 64, dtype=torch.bfloat16) * 2
    plan = attn.DecodePlan(pg.cache, 16, len(lens))
    got = plan.run(q, pg.table, pg.len_t)
    o, w = pg.want(q, 64 ** -0.5)
    close(got, o, w)
    for _ in range(3):  # the split is joined in a fixed order, and the workspace left as it was
        assert torch.equal(plan.run(q, pg.table, pg.len_t), got)


@pytest.mark.parametrize("hq,hk,d,page,e4m3", [(16, 2, 64, 16, True), (24, 2, 128, 48, False), (4, 4, 128, 16, True),
                                               (6, 1, 64, 32, False)])
def test_decode_many_ragged(hq, hk, d, page, e4m3):
    """Hundreds of sequences, many empty or short, some cut between warps and blocks."""
    g = gen(hq + page)
    r = torch.Generator().manual_seed(page)
    lens = [int(x) for x in (700 * torch.rand(400, generator=r) ** 4)]
    lens[17] = 9000
    lens[399] = 0
    pg = Paged(g, lens, hk, d, page, e4m3)
    q = randn(g, len(lens), hq, d, dtype=torch.bfloat16) * 2
    plan = attn.DecodePlan(pg.cache, hq, len(lens))
    got = plan.run(q, pg.table, pg.len_t)
    close(got, *pg.want(q, d ** -0.5))
    for _ in range(2):
        assert torch.equal(plan.run(q, pg.table, pg.len_t), got)
    attn.check()


@pytest.mark.parametrize("lens", [[61] * 28, [32] * 101, [7 * i % 119 for i in range(112)], [496] * 21, [1] * 148])
@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_many_short(lens, e4m3):
    """More short items than blocks: four, two or one warp each, none cut between blocks."""
    g = gen(len(lens) + e4m3)
    pg = Paged(g, lens, 8, 128, 32, e4m3)
    q = randn(g, len(lens), 16, 128, dtype=torch.bfloat16) * 2
    plan = attn.DecodePlan(pg.cache, 16, len(lens))
    got = plan.run(q, pg.table, pg.len_t)
    close(got, *pg.want(q, 128 ** -0.5))
    assert torch.equal(plan.run(q, pg.table, pg.len_t), got)
    attn.check()


@pytest.mark.parametrize("hk,d,e4m3", [(1, 64, False), (1, 128, True), (2, 128, False)])
def test_decode_one_item_over_all_blocks(hk, d, e4m3):
    """Few pairs on a long cache: partials of up to all blocks joined, groups of 8 and of 16 heads."""
    for hq in (8 * hk, 16 * hk):
        g = gen(hk + d + hq)
        pg = Paged(g, [50021], hk, d, 64, e4m3)
        q = randn(g, 1, hq, d, dtype=torch.bfloat16) * 2
        plan = attn.DecodePlan(pg.cache, hq, 1)
        got = plan.run(q, pg.table, pg.len_t)
        close(got, *pg.want(q, d ** -0.5))
        assert torch.equal(plan.run(q, pg.table, pg.len_t), got)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("peak", [1e-3, 12.0, 60.0])
def test_decode_flat_and_peaked_scores(peak, e4m3):
    """Scores from all alike to one key taking all; the largest near the start, middle and end."""
    g = gen(int(peak) + 5)
    lens = [2000, 2000, 2000, 40]
    pg = Paged(g, lens, 1, 128, 64, e4m3)
    q = randn(g, 4, 8, 128, dtype=torch.bfloat16)
    for b, at in enumerate((0, 1000, 1999, 39)):
        q[b] = (q[b].double() * 0.1 + pg.rows[b][0][at, 0] * peak / 11.3).to(torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 8, 4)
    got = plan.run(q, pg.table, pg.len_t)
    o, w = pg.want(q, 128 ** -0.5)
    close(got, o, w)


@pytest.mark.parametrize("big", [1e30, 3e38])
def test_decode_huge_queries_on_e4m3(big):
    """q beyond the range of 16-bit floats with small exponents; a tiny scale brings the scores back."""
    g = gen(11)
    pg = Paged(g, [200, 33], 1, 128, 64, True)
    unit = randn(g, 2, 8, 128).clamp(-1, 1)
    q = (unit * big).to(torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 8, 2, scale=float(1.0 / big))
    got = plan.run(q, pg.table, pg.len_t)
    o, w = pg.want(q, float(torch.tensor(1.0 / big, dtype=torch.float32)))
    close(got, o, w)


def test_decode_many_small_weights_on_e4m3():
    """One key of score 17.3 among 200,000 of score 0, whose weights of 2^-25 sum up to the result."""
    n, d = 200000, 128
    cache = attn.KvCache.empty(n // 64, 1, 64, d, E4M3)
    k = torch.zeros((n, d), device="cuda")
    v = torch.ones((n, d), device="cuda")
    k[777], v[777] = 1.0, 0.0
    cache.k.copy_(k.view(-1, 1, 64, d).to(E4M3))
    cache.v.copy_(v.view(-1, 1, 64, d).to(E4M3))
    q = torch.ones((1, 8, d), device="cuda", dtype=torch.bfloat16)
    scale = 17.3 / d
    got = attn.DecodePlan(cache, 8, 1, scale=scale).run(
        q, torch.arange(n // 64, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda"))
    o, w = softmax_rows(q[0], k, v, scale, torch.ones(8, n, dtype=torch.bool, device="cuda"))
    assert 5e-3 < float(o[0, 0]) < 7e-3
    close(got[0], o, w)


def test_calls_work_after_shutdown_and_init():
    """Set-up per device is done again after colizig_cuda_shutdown; the caller's buffers stay good."""
    g = gen(50)
    pg = Paged(g, [300, 20], 2, 128, 64)
    q = randn(g, 2, 8, 128, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 8, 2)
    want = plan.run(q, pg.table, pg.len_t)
    pq, pk, pv, cu = prompts(g, [200], [200], 8, 2, 128, False)
    wantp = attn.prefill(pq, pk, pv, cu[0])
    torch.cuda.synchronize()
    gpu.deinit()
    gpu.init()
    assert torch.equal(plan.run(q, pg.table, pg.len_t), want)
    assert torch.equal(attn.prefill(pq, pk, pv, cu[0]), wantp)
    attn.check()


def test_decode_offsets_past_32_bits():
    """Pages whose first element lies past 2^32."""
    page, hk, d = 64, 1, 128
    pages = (1 << 32) // (page * hk * d) + 40
    k = torch.zeros((pages, hk, page, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(3)
    rows = [pages - 1, 0, pages - 20, pages // 2 + 3]
    x = randn(g, 2, len(rows) * page, d, dtype=torch.bfloat16)
    for i, r in enumerate(rows):
        k[r, 0], v[r, 0] = x[0, i * page:(i + 1) * page], x[1, i * page:(i + 1) * page]
    table = torch.tensor([rows], dtype=torch.int32, device="cuda")
    n = len(rows) * page - 5
    q = randn(g, 1, 8, d, dtype=torch.bfloat16)
    cache = attn.KvCache(k, v)
    got = attn.DecodePlan(cache, 8, 1).run(q, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    o, w = softmax_rows(q[0], x[0][:n], x[1][:n], d ** -0.5, torch.ones(8, n, dtype=torch.bool, device="cuda"))
    close(got[0], o, w)
    # append to the far pages
    T = 3
    slots = torch.tensor([(pages - 1) * page + 63, 5, (pages - 20) * page], device="cuda")
    kv = randn(g, 2, T, hk, d, dtype=torch.bfloat16)
    attn.append(cache, randn(g, T, 8, d, dtype=torch.bfloat16), kv[0], kv[1], None, slots)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k[s // page, 0, s % page], kv[0, i, 0]) and torch.equal(v[s // page, 0, s % page], kv[1, i, 0])
    attn.check()


def test_decode_bad_indices_are_reported_and_not_followed():
    g = gen(4)
    pg = Paged(g, [100, 90, 64, 10], 2, 128, 32)
    q = randn(g, 4, 4, 128, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 4, 4)
    good = plan.run(q, pg.table, pg.len_t)
    attn.check()
    for bad in (pg.cache.pages, -1, 2 ** 31 - 1, -2 ** 31):
        table = pg.table.clone()
        table[0, 1] = bad
        got = plan.run(q, table, pg.len_t)
        assert torch.equal(got[1:], good[1:])
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11
        attn.check()  # cleared
    for n in (pg.width * 32 + 1, -1, 2 ** 31 - 1, -2 ** 31):
        lens = pg.len_t.clone()
        lens[1] = n
        got = plan.run(q, pg.table.clamp(min=0), lens)
        assert torch.equal(got[0], good[0]) and torch.equal(got[2:], good[2:])
        with pytest.raises(ColizigError):
            attn.check()
    assert torch.equal(plan.run(q, pg.table, pg.len_t), good)
    attn.check()


@pytest.mark.parametrize("at", [0, 33, 150, 199])
def test_decode_bad_length_in_a_large_batch(at):
    g = gen(60)
    pg = Paged(g, [5 + i % 40 for i in range(200)], 1, 64, 16)
    q = randn(g, 200, 2, 64, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 2, 200)
    good = plan.run(q, pg.table, pg.len_t)
    attn.check()
    for bad in (-3, pg.width * 16 + 1):
        lens = pg.len_t.clone()
        lens[at] = bad
        got = plan.run(q, pg.table.clamp(min=0), lens)
        keep = torch.arange(200, device="cuda") != at
        assert torch.equal(got[keep], good[keep])
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11


def test_prefill_bad_bounds_among_many_are_reported():
    g = gen(61)
    n = [3 + i % 20 for i in range(90)]
    q, k, v, cu = prompts(g, n, n, 4, 2, 64, False)
    good = attn.prefill(q, k, v, cu[0])
    attn.check()
    for at in (1, 40, 90):
        bad = cu[1].clone()
        bad[at] = k.shape[0] + 7
        got = attn.prefill(q, k, v, cu[0], bad)
        rows = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
        ends = cu[0].tolist()
        rows[ends[at - 1]: ends[min(at + 1, 90)]] = False  # the sequences that name the bad bound
        assert torch.equal(got[rows], good[rows])
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11


def test_decode_in_a_graph_follows_lengths():
    """Lengths and tables are read on the device: one captured step serves a growing cache."""
    g = gen(5)
    pg = Paged(g, [400, 800, 3], 2, 128, 64)
    q = randn(g, 3, 16, 128, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 16, 3)
    lens = pg.len_t.clone()
    out = plan.run(q, pg.table, lens)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        plan.run(q, pg.table, lens, out=out)
    for cut in ([400, 800, 3], [1, 799, 0], [64, 65, 2], [400, 128, 1]):
        lens.copy_(torch.tensor(cut, dtype=torch.int32))
        out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        full, pg.lens = pg.lens, cut
        rows, pg.rows = pg.rows, [r[:, :n] for r, n in zip(pg.rows, cut)]
        o, w = pg.want(q, 128 ** -0.5)
        pg.lens, pg.rows = full, rows
        close(out, o, w)


# ------------------------------------------------------------------ prefill


def prompts(g, nq, nk, hq, hk, d, fused):
    tq, tk = sum(nq), sum(nk)
    if fused:
        row = (hq + 2 * hk) * d + 24
        buf = torch.full((max(tq, tk), row), NAN, device="cuda", dtype=torch.bfloat16)
        q = buf[:tq, : hq * d].unflatten(1, (hq, d))
        k = buf[:tk, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
        v = buf[:tk, (hq + hk) * d: (hq + 2 * hk) * d].unflatten(1, (hk, d))
    else:
        q, k, v = (torch.empty(s, device="cuda", dtype=torch.bfloat16) for s in ((tq, hq, d), (tk, hk, d), (tk, hk, d)))
    q.copy_(randn(g, tq, hq, d) * 2)
    k.copy_(randn(g, tk, hk, d))
    v.copy_(randn(g, tk, hk, d))
    cu = [torch.tensor([0] + list(x), dtype=torch.int32).cumsum(0).int().cuda() for x in (nq, nk)]
    return q, k, v, cu


def prefill_want(q, k, v, nq, nk, scale):
    hq, hk = q.shape[1], k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    w = torch.zeros_like(o)
    a = b = 0
    for i, j in zip(nq, nk):
        seen = torch.ones(i, j, dtype=torch.bool, device="cuda").tril(j - i)
        for h in range(hq):
            if i and j:
                r = softmax_rows(q[a:a + i, h], k[b:b + j, h * hk // hq], v[b:b + j, h * hk // hq], scale, seen)
                o[a:a + i, h], w[a:a + i, h] = r
        a, b = a + i, b + j
    return o, w


RAGGED = [1, 0, 2, 15, 16, 17, 31, 33, 127, 128, 129, 64, 255, 257, 3]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 128), (32, 4, 128), (4, 4, 64), (3, 3, 128), (10, 2, 128), (14, 2, 64),
                                     (6, 1, 128), (24, 2, 64), (16, 1, 128), (33, 1, 128), (128, 1, 64), (130, 1, 64)])
def test_prefill_head_layouts(hq, hk, d, fused):
    g = gen(hq + hk + d)
    q, k, v, cu = prompts(g, RAGGED, RAGGED, hq, hk, d, fused)
    got = attn.prefill(q, k, v, cu[0])
    close(got, *prefill_want(q, k, v, RAGGED, RAGGED, d ** -0.5))
    attn.check()


@pytest.mark.parametrize("d", [64, 128])
def test_prefill_keys_before_and_rows_that_see_none(d):
    nq = [5, 130, 1, 40, 7, 300, 0, 64, 9]
    nk = [900, 131, 257, 3, 0, 299, 12, 64, 640]  # 40 queries on 3 keys, 7 on none, 300 on 299
    g = gen(d)
    q, k, v, cu = prompts(g, nq, nk, 8, 2, d, True)
    got = attn.prefill(q, k, v, cu[0], cu[1], scale=0.2)
    o, w = prefill_want(q, k, v, nq, nk, 0.2)
    close(got, o, w)
    none = torch.cat([(torch.arange(i) + j - i < 0) for i, j in zip(nq, nk)]).cuda()
    assert int(none.sum()) == 37 + 7 + 1 and not got[none].any()


def test_prefill_of_nothing_and_of_no_keys():
    q = torch.empty((0, 8, 128), device="cuda", dtype=torch.bfloat16)
    cu0 = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert attn.prefill(q, q[:, :2], q[:, :2], cu0).shape == (0, 8, 128)
    q = torch.full((4, 8, 128), 1.0, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 4, 4], dtype=torch.int32, device="cuda")
    kv = torch.empty((0, 2, 128), device="cuda", dtype=torch.bfloat16)
    assert not attn.prefill(q, kv, kv, cu, cu0).any()


def test_prefill_many_prompts():
    """Several rounds of query tiles per block, more sequences than a warp has lanes."""
    r = torch.Generator().manual_seed(1)
    nq = [int(x) for x in 500 * torch.rand(150, generator=r) ** 3]
    nk = [n + (37 * i % 300 if i % 4 == 0 else 0) for i, n in enumerate(nq)]
    g = gen(8)
    q, k, v, cu = prompts(g, nq, nk, 6, 2, 64, False)
    got = attn.prefill(q, k, v, *cu)
    close(got, *prefill_want(q, k, v, nq, nk, 64 ** -0.5))
    assert torch.equal(attn.prefill(q, k, v, *cu), got)
    attn.check()


@pytest.mark.parametrize("n", [1024, 2500, 4099])
def test_prefill_long_prompt(n):
    g = gen(n)
    q, k, v, cu = prompts(g, [n], [n], 8, 1, 128, False)
    got = attn.prefill(q, k, v, cu[0])
    close(got, *prefill_want(q, k, v, [n], [n], 128 ** -0.5))
    assert torch.equal(attn.prefill(q, k, v, cu[0]), got)


@pytest.mark.parametrize("peak", [1e-3, 12.0, 60.0])
def test_prefill_flat_and_peaked_scores(peak):
    """Rows whose largest score moves up late (keys growing along the prompt) and early."""
    g = gen(9)
    n = 700
    q, k, v, cu = prompts(g, [n, n], [n, n], 4, 2, 128, False)
    ramp = torch.linspace(0.1, 1, n, device="cuda")[:, None, None]
    k[:n] = (k[:n].float() * ramp).bfloat16()
    k[n:] = (k[n:].float() * ramp.flip(0)).bfloat16()
    q.copy_(q.float() * (peak / 12))
    got = attn.prefill(q, k, v, cu[0])
    close(got, *prefill_want(q, k, v, [n, n], [n, n], 128 ** -0.5))


def test_prefill_neighbours_never_leak():
    """NaN and infinity in one sequence's rows stay out of the others' results."""
    g = gen(21)
    nq = [100, 50, 100]
    for bad in (NAN, math.inf):
        q, k, v, cu = prompts(g, nq, nq, 8, 2, 128, True)
        for t in (q, k, v):
            t[100:150] = bad
        got = attn.prefill(q, k, v, cu[0])
        q, k, v = q.clone(), k.clone(), v.clone()
        for t in (q, k, v):
            t[100:150] = 0
        o, w = prefill_want(q, k, v, nq, nq, 128 ** -0.5)
        close(got[:100], o[:100], w[:100])
        close(got[150:], o[150:], w[150:])


def test_prefill_bad_bounds_are_reported_and_not_followed():
    g = gen(22)
    q, k, v, cu = prompts(g, [60, 60], [60, 60], 4, 2, 128, False)
    good = attn.prefill(q, k, v, cu[0])
    attn.check()
    for bad in ([0, 60, 2 ** 31 - 1], [0, 60, 121], [0, -5, 120], [0, 130, 120], [-7, 60, 120]):
        b = torch.tensor(bad, dtype=torch.int32, device="cuda")
        attn.prefill(q, k, v, cu[0], b)
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11
        attn.prefill(q, k, v, b, cu[1])
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11
    assert torch.equal(attn.prefill(q, k, v, cu[0]), good)
    attn.check()


# ------------------------------------------------------------------ append


def heads_want(x, w, rope, positions, eps):
    """(y, length of the rotated pair or |y|) in f64."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs()
    if rope is not None:
        r = rope.shape[1]
        c, s = (t[:, None] for t in rope.double()[positions.long()].split(r // 2, 1))
        a, b = y[..., : r // 2], y[..., r // 2: r]
        pair = (a.square() + b.square()).sqrt()
        y = torch.cat([a * c - b * s, b * c + a * s, y[..., r:]], -1)
        size = torch.cat([pair, pair, size[..., r:]], -1)
    return y, size


def within(got, want, size, step, floor=0.0):
    got = got.double()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - (want.abs() * step + size * 2.0 ** -20 + floor)
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("x", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d,rot,norm,T,page", [(32, 4, 128, 128, True, 1, 64), (32, 4, 128, 128, True, 77, 16),
                                                     (6, 2, 64, 64, False, 130, 48), (16, 16, 64, 32, True, 33, 128),
                                                     (5, 1, 128, 64, True, 50, 64), (7, 7, 128, 16, False, 9, 32),
                                                     (4, 4, 64, 0, True, 20, 64), (64, 8, 128, 112, False, 300, 64),
                                                     (16, 16, 64, 64, True, 900, 32)])
def test_append(hq, hk, d, rot, norm, T, page, x, e4m3):
    g = gen(T + hq)
    eps = 1e-5
    row = (hq + 2 * hk) * d + 8
    qkv = randn(g, T, row, dtype=x) * 3
    q = qkv[:, : hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
    v = qkv[:, (hq + hk) * d: (hq + 2 * hk) * d].unflatten(1, (hk, d))
    pages = T // page + 3
    ks = vs = None
    dtype = torch.bfloat16
    if e4m3:
        dtype = E4M3
        ks = 0.02 + 0.05 * torch.rand(hk, generator=g, device="cuda")
        vs = 0.005 + 0.05 * torch.rand(hk, generator=g, device="cuda")  # some values saturate
    cache = attn.KvCache.empty(pages, hk, page, d, dtype, k_scale=ks, v_scale=vs)
    before = 0x33
    cache.k.view(torch.uint8).fill_(before)
    cache.v.view(torch.uint8).fill_(before)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T].cuda()
    slots[T // 2::5] = -1 if T > 3 else slots[T // 2::5]
    positions = torch.randint(0, 100000, (T,), generator=g, device="cuda", dtype=torch.int32)
    positions[0] = 99999
    rope = attn.rope_table(100000, rot) if rot else None
    qn = 1 + 0.3 * randn(g, d) if norm else None
    kn = 1 + 0.3 * randn(g, d) if norm else None
    gq, gk, gv = attn.append(cache, q, k, v, positions if rot else None, slots, rope, qn, kn, eps, packed=True)
    wq, sq = heads_want(q, qn, rope, positions, eps)
    wk, sk = heads_want(k, kn, rope, positions, eps)
    within(gq, wq, sq, 2.0 ** -8)
    within(gk, wk, sk, 2.0 ** -8)
    assert torch.equal(gv, v.bfloat16())
    touched = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    kept = slots >= 0
    touched[slots[kept]] = True
    for got, want, size, sc in ((cache.k, wk, sk, ks), (cache.v, v.double(), v.double().abs(), vs)):
        flat = got.view(torch.uint8).transpose(1, 2).reshape(pages * page, -1)
        assert (flat[~touched] == before).all()  # nothing else is written
        at = flat[slots[kept]].contiguous().view(dtype).view(-1, hk, d)
        if e4m3:
            s = sc.double()[:, None]
            top = 448 * s
            within(at.double() * s, want[kept].clamp(-top, top), size[kept], 2.0 ** -4, s * 2.0 ** -10)
        else:
            within(at, want[kept], size[kept], 2.0 ** -8)
    attn.check()
    # the same call without the packed copies
    assert attn.append(cache, q, k, v, positions if rot else None, slots, rope, qn, kn, eps)[1:] == (None, None)


def test_append_special_values():
    """Zero rows under the norm, infinities and NaN stay in their own head and token."""
    g = gen(2)
    T, hq, hk, d = 6, 4, 2, 128
    q, k, v = randn(g, T, hq, d), randn(g, T, hk, d), randn(g, T, hk, d)
    q[0] = 0
    q[1, 2] = NAN
    k[2, 0, 5] = math.inf
    v[3, 1, 7] = -math.inf
    w = torch.ones(d, device="cuda")
    rope = attn.rope_table(8, 64)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    for dtype in (torch.bfloat16, E4M3):
        cache = attn.KvCache.empty(1, hk, 16, d, dtype)
        gq, gk, gv = attn.append(cache, q, k, v, pos, torch.arange(T, device="cuda"), rope, w, w, packed=True)
        assert not gq[0].any() and gq[1, 2].isnan().all()
        fine = torch.ones(T, hq, dtype=torch.bool, device="cuda")
        fine[1, 2] = False
        assert torch.isfinite(gq[fine]).all()
        fine = torch.ones(T, hk, dtype=torch.bool, device="cuda")
        fine[2, 0] = False
        assert torch.isfinite(gk[fine]).all()
        assert gv[3, 1, 7] == -math.inf and int((~torch.isfinite(gv)).sum()) == 1
        cv = cache.v[0].transpose(0, 1).float()[:T]
        assert cv[3, 1, 7] == (-math.inf if dtype == torch.bfloat16 else -448)
        assert torch.isfinite(cv).sum() == cv.numel() - (dtype == torch.bfloat16)


def test_append_bad_indices_are_reported_and_not_followed():
    g = gen(6)
    T, hk, d = 4, 2, 128
    q, k, v = randn(g, T, 4, d), randn(g, T, hk, d), randn(g, T, hk, d)
    rope = attn.rope_table(16, d)
    cache = attn.KvCache.empty(2, hk, 16, d)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    good = torch.arange(T, device="cuda")
    attn.append(cache, q, k, v, pos, good, rope)
    attn.check()
    k0 = cache.k.clone()
    for bad in (32, 2 ** 40, 2 ** 63 - 1):
        s = good.clone()
        s[2] = bad
        attn.append(cache, q, k, v, pos, s, rope)
        assert torch.equal(cache.k, k0)
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11
    for bad in (16, -1, 2 ** 31 - 1, -2 ** 31):
        p = pos.clone()
        p[1] = bad
        attn.append(cache, q, k, v, p, good, rope)
        with pytest.raises(ColizigError) as e:
            attn.check()
        assert e.value.rc == -11
    s = good.clone()
    s[3] = -2 ** 63  # negative: not cached, no error
    attn.append(cache, q, k, v, pos, s, rope)
    attn.check()


def test_append_of_no_tokens():
    cache = attn.KvCache.empty(1, 2, 16, 128)
    e = torch.empty((0, 2, 128), device="cuda")
    q, k, v = attn.append(cache, e, e, e, None, torch.empty(0, dtype=torch.int64, device="cuda"), packed=True)
    assert q.shape == (0, 2, 128) and k.shape == (0, 2, 128)


# ------------------------------------------------------------------ together


def test_append_decode_and_prefill_agree():
    """A prompt through prefill gives what decode gives when its tokens come one by one."""
    g = gen(33)
    T, hq, hk, d, page = 70, 32, 4, 128, 16
    cache = attn.KvCache.empty(8, hk, page, d)
    rope = attn.rope_table(T, d)
    w = 1 + 0.1 * randn(g, d)
    q, k, v = randn(g, T, hq, d), randn(g, T, hk, d), randn(g, T, hk, d)
    order = torch.tensor([5, 2, 7, 0, 3], device="cuda")
    i = torch.arange(T, device="cuda")
    slots = order[i // page] * page + i % page
    pq, pk, pv = attn.append(cache, q, k, v, i.int(), slots, rope, w, w, packed=True)
    whole = attn.prefill(pq, pk, pv, torch.tensor([0, T], dtype=torch.int32, device="cuda"))
    plan = attn.DecodePlan(cache, hq, T)
    steps = plan.run(pq, order.int().expand(T, -1).contiguous(), (i + 1).int())
    # two roundings of the same value, and the weights' roundings: twice a call's own tolerance
    o, s = prefill_want(pq, pk, pv, [T], [T], d ** -0.5)
    close(whole, o, s)
    close(steps, o, s)


def test_other_streams():
    """Calls queued on a given stream are ordered there and nowhere else; so are their outputs."""
    g = gen(40)
    pg = Paged(g, [500, 77], 4, 128, 64)
    q = randn(g, 2, 32, 128, dtype=torch.bfloat16)
    plan = attn.DecodePlan(pg.cache, 32, 2)
    want = plan.run(q, pg.table, pg.len_t)
    pq, pk, pv, cu = prompts(g, [100], [100], 8, 2, 128, False)
    wantp = attn.prefill(pq, pk, pv, cu[0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(5):
        q2 = torch.zeros_like(q)
        pq2 = torch.zeros_like(pq)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
            q2.copy_(q)
            pq2.copy_(pq)
        got = plan.run(q2, pg.table, pg.len_t, stream=s)
        gotp = attn.prefill(pq2, pk, pv, cu[0], stream=s.cuda_stream)
        del q2, pq2  # their memory may not be reused before the calls are done
        junk = [torch.full_like(q, NAN) for _ in range(4)] + [torch.full_like(pq, NAN) for _ in range(4)]
        s.synchronize()
        assert torch.equal(got, want) and torch.equal(gotp, wantp)
        del junk


# ------------------------------------------------------------------ refusals


def test_refusals():
    gpu.init()
    bf = torch.bfloat16
    kv = torch.zeros((4, 2, 16, 128), dtype=bf, device="cuda")
    for k, v, kw in [
        (kv, kv[:3], {}), (kv, kv.float(), {}), (kv.float(), kv.float(), {}), (kv.cpu(), kv.cpu(), {}),
        (kv[..., :96], kv[..., :96], {}), (kv[:, :, :8], kv[:, :, :8], {}), (kv[:0], kv[:0], {}),
        (kv.transpose(1, 2), kv.transpose(1, 2), {}), (kv, kv, {"k_scale": torch.ones(2, device="cuda")}),
        (kv.to(E4M3), kv.to(E4M3), {"v_scale": torch.ones(3, device="cuda")}),
        (kv.to(E4M3), kv.to(E4M3), {"v_scale": torch.ones(2, device="cuda", dtype=torch.float64)}),
        (kv.view(-1)[1:-15].view(-1)[: 3 * 4096].view(3, 2, 16, 128),) * 2 + ({},),
    ]:
        with pytest.raises(ValueError):
            attn.KvCache(k, v, **kw)
    cache = attn.KvCache(kv, kv.clone())
    for hq, b in ((3, 1), (0, 1), (4, 0), (4, 5000)):
        with pytest.raises(ValueError):
            attn.DecodePlan(cache, hq, b)
    plan = attn.DecodePlan(cache, 4, 2)
    q = torch.zeros((2, 4, 128), dtype=bf, device="cuda")
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    plan.run(q, table, lens)
    for a in [(q.float(), table, lens), (q[:, :2], table, lens), (q.transpose(1, 2), table, lens),
              (q, table.long(), lens), (q, table[:1], lens), (q, table, lens.long()), (q, table, lens[:1]),
              (q, table[:, :0], lens), (q.cpu(), table, lens), (q, table.cpu(), lens), (q, table, lens.cpu()),
              (torch.zeros((3, 4, 128), dtype=bf, device="cuda"), table, lens),
              (q, torch.zeros((3, 2), dtype=torch.int32, device="cuda").T, lens),
              (q, table, lens, q.float()), (q, table, lens, q[:1])]:
        with pytest.raises(ValueError):
            plan.run(*a)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    k = torch.zeros((2, 2, 128), dtype=bf, device="cuda")
    attn.prefill(q, k, k, cu)
    for a in [(q.float(), k, k, cu), (q, k[:, :1], k, cu), (q, k[:1], k[:1], cu), (q[..., :64], k, k, cu),
              (q[:, :3], k, k, cu), (q, k, k[:1], cu, cu), (q, k, k, cu.long()), (q, k, k, cu, cu[:1]),
              (q, k, k, cu[:0]), (q, k, k, cu.cpu()), (q.cpu(), k, k, cu), (q, k.transpose(1, 2), k, cu)]:
        with pytest.raises(ValueError):
            attn.prefill(*a)
    slots = torch.zeros(2, dtype=torch.int64, device="cuda") - 1
    rope = attn.rope_table(4, 128)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    attn.append(cache, q, k, k, pos, slots, rope)
    for a, kw in [((q, k, k.float(), pos, slots, rope), {}), ((q.half(), k, k, pos, slots, rope), {}),
                  ((q[:1], k, k, pos, slots, rope), {}), ((q[:, :3], k, k, pos, slots, rope), {}),
                  ((q, k, k, pos, slots.int(), rope), {}), ((q, k, k, pos.long(), slots, rope), {}),
                  ((q, k, k, pos, slots[:1], rope), {}), ((q, k, k, pos[:1], slots, rope), {}),
                  ((q, k, k, pos, slots, rope[:, :24]), {}), ((q, k, k, pos, slots, rope.double()), {}),
                  ((q, k, k, pos, slots, rope), {"q_norm": torch.ones(64, device="cuda")}),
                  ((q, k, k, pos, slots, rope), {"k_norm": torch.ones(128, device="cuda", dtype=bf)}),
                  ((q, k, k, pos, slots, rope), {"k_norm": torch.ones(129, device="cuda")[1:]}),
                  ((q, k, k, pos, slots, rope), {"q_out": q.float()}),
                  ((q, k, k, pos, slots, rope), {"k_out": q})]:
        with pytest.raises(ValueError):
            attn.append(cache, *a, **kw)


def test_refusals_of_the_c_entry_points():
    """The library checks what a caller of the C interface may get wrong; nothing is launched."""
    import ctypes

    from colizig_b200 import _abi

    gpu.init()
    L = _abi.load()
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    P = t.data_ptr()

    def kv(**kw):
        d = dict(k=P, v=P, k_scale=None, v_scale=None, k_page_stride=4096, v_page_stride=4096, pages=2, page_size=16,
                 kv_heads=2, head_dim=128, dtype=0)
        d.update(kw)
        return ctypes.byref(_abi.KvCacheC(**d))

    dec = dict(c=None, q=P, qs=512, B=1, hq=4, t=P, w=1, ts=1, l=P, s=1.0, o=P, ws=P, st=None)

    def decode(**kw):
        d = dict(dec, c=kv())
        d.update(kw)
        return L.colizig_cuda_attn_decode(*d.values())

    assert decode(B=0) == 0
    for bad in ({"k": None}, {"v": P + 8}, {"dtype": 2}, {"k_page_stride": 4095}, {"v_page_stride": 4097},
                {"k_scale": P}):
        assert decode(c=kv(**bad)) == -1, bad
    for bad in ({"pages": 0}, {"page_size": 8}, {"page_size": 24}, {"head_dim": 96}, {"kv_heads": 0},
                {"page_size": 1 << 20}):
        assert decode(c=kv(**bad)) == -8, bad
    for kw, rc in (({"c": None}, -1), ({"q": None}, -1), ({"q": P + 2}, -1), ({"t": None}, -1), ({"l": None}, -1),
                   ({"o": None}, -1), ({"o": P + 4}, -1), ({"ws": None}, -1), ({"ws": P + 16}, -1), ({"w": 0}, -1),
                   ({"ts": 0}, -1), ({"qs": 511}, -1), ({"qs": 516}, -1), ({"B": -1}, -1), ({"B": 4097}, -8),
                   ({"hq": 3}, -8), ({"hq": 0}, -8), ({"w": 1 << 30, "ts": 1 << 30}, -8)):
        assert decode(**kw) == rc, kw
    pre = dict(q=P, k=P, v=P, qs=512, ks=256, vs=256, Tq=2, Tk=2, B=1, hq=4, hk=2, d=128, cq=P, ck=P, s=1.0, o=P, st=None)

    def prefill(**kw):
        d = dict(pre)
        d.update(kw)
        return L.colizig_cuda_attn_prefill(*d.values())

    for kw, rc in (({"Tq": 0}, 0), ({"B": 0}, 0), ({"Tq": -1}, -1), ({"q": None}, -1), ({"k": None}, -1),
                   ({"v": P + 8}, -1), ({"qs": 504}, -1), ({"ks": 260}, -1), ({"vs": 128}, -1), ({"cq": None}, -1),
                   ({"ck": None}, -1), ({"o": None}, -1), ({"d": 32}, -8), ({"hq": 5}, -8), ({"hk": 0}, -8),
                   ({"B": 5000}, -8)):
        assert prefill(**kw) == rc, kw
    ap = dict(c=None, q=P, k=P, v=P, xd=1, T=1, hq=4, qs=512, ks=256, vs=256, p=P, s=P, r=P, rl=1, rd=128, qn=None,
              kn=None, e=1e-6, qo=P, ko=None, vo=None, st=None)

    def append(**kw):
        d = dict(ap, c=kv())
        d.update(kw)
        return L.colizig_cuda_attn_append(*d.values())

    for kw, rc in (({"T": 0}, 0), ({"T": -1}, -1), ({"xd": 2}, -1), ({"q": None}, -1), ({"k": P + 2}, -1),
                   ({"s": None}, -1), ({"qo": None}, -1), ({"r": None}, -1), ({"p": None}, -1), ({"rl": 0}, -1),
                   ({"rd": 0}, -1), ({"rd": 24}, -8), ({"rd": 144}, -8), ({"hq": 5}, -8), ({"qs": 500}, -1),
                   ({"ks": 252}, -1), ({"vs": 260}, -1), ({"ko": P + 8}, -1), ({"qn": P + 4}, -1),
                   ({"xd": 0, "qs": 514}, -1)):
        assert append(**kw) == rc, kw
    torch.cuda.synchronize()
