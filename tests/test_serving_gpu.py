"""GPU tests of the paged 4-bit serving operators against 64-bit restatements
(oracle/serving.py): page plan, quantised write and read, the quantising new-token
preparation, attention over the 4-bit pages, per-request low-rank adapters.

Integers, cache bytes and dequantised values are compared exactly: quantisation is defined
bit for bit, and every value it yields has at most 8 significant bits.

Tolerances of the computed outputs, from their roundings:
  attention  |err| <= (2^-9 + 2^-9 + 2 d) sum_s p_s |v_s|: the stored probabilities (at most
             bf16's 2^-9), the bf16 output (its size is at most that sum), and scores whose
             fp32 sums of 576 products are off by d = 576 * 2^-24 * max sum |q k| * scale, which
             changes every p by at most a factor e^(2 d); 2^-7 leaves room for both factors
             above 1 + d and for the fp32 sums over positions
  adapters   |err| <= 2^-8 |y| + 2^-8 sum_j |low_j B_j| + K 2^-23 sum |x w|: the bf16 output,
             the low-rank activations in at least bf16, fp32 sums of K products
"""
import math

import pytest
import torch

from oracle import serving as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def D():
    from dsv2 import _lib, ops
    _lib.load()
    _lib.device_error(clear=True)
    return ops


@pytest.fixture(autouse=True)
def no_device_error():
    from dsv2 import _lib
    _lib.device_error(clear=True)
    yield
    assert _lib.device_error(clear=True) == 0


def expect_error(code):
    from dsv2 import _lib
    assert _lib.device_error(clear=True) == code


def rows_of(n, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, 576, generator=g) * scale).to(torch.bfloat16)


# ------------------------------------------------------------------ page plan
def plan_case(R, page, width, free, seed, capacity, finish=True, big=0):
    g = torch.Generator().manual_seed(seed)
    most = width * page
    cached = torch.randint(0, max(1, most // 2), (R,), generator=g)
    cached[torch.rand(R, generator=g) < 0.1] = 0
    new = torch.randint(0, 3, (R,), generator=g)
    if big and R:
        new[torch.randint(0, R, (max(1, R // 8),), generator=g)] = big
    if finish:
        new[torch.rand(R, generator=g) < 0.15] = -1
    held = (cached + page - 1) // page
    total = int(held.sum()) + free
    size = total + 5
    pages = torch.randperm(size, generator=g)
    table = torch.full((R, width), -7, dtype=torch.int64)
    at = 0
    for r in range(R):
        table[r, :held[r]] = pages[at:at + held[r]]
        at += int(held[r])
    ring = torch.full((size,), -9, dtype=torch.int64)
    head = 3 * size + size // 2 + 1                       # the ring has been round a few times
    for i in range(free):
        ring[(head + i) % size] = pages[at + i]
    return cached, new, table, ring, (head, head + free), page, capacity


def run_plan(D, case, alias=False, cached_dtype=torch.int32, stride=None):
    cached, new, table, ring, (head, tail), page, cap = case
    R, width = table.shape
    buf = D.page_plan_buffers(R, cap, DEV)
    for v in buf.values():
        if v is not buf["sync"]:
            v.fill_(-99)
    wide = torch.full((R, stride or width), -3, dtype=torch.int32, device=DEV)
    wide[:, :width] = table.to(DEV, torch.int32)
    tab = wide[:, :width]
    rin = torch.tensor([head, tail], dtype=torch.int64, device=DEV)
    if alias:
        buf["ring_out"] = rin
    rg = ring.to(DEV, torch.int32)
    D.page_plan(cached=cached.to(DEV, cached_dtype), new=new.to(DEV, torch.int32), block_table=tab, free_ring=rg,
                ring_in=rin, page_size=page, **buf)
    torch.cuda.synchronize()
    assert int(buf["sync"]) == 0
    if stride:
        assert bool((wide[:, width:] == -3).all())
    return {**{k: v.cpu().tolist() for k, v in buf.items() if k != "sync"}, "table": tab.cpu().tolist(), "ring": rg.cpu().tolist()}


def want_plan(case):
    cached, new, table, ring, rin, page, cap = case
    t, rg = table.tolist(), ring.tolist()
    out = S.page_plan(cached.tolist(), new.tolist(), t, rg, rin, page, cap)
    return {**out, "table": t, "ring": rg}


# requests around the chunk of 1024, capacities around the group of 1024 token rows, enough free
# pages and too few, every page-size kind
@pytest.mark.parametrize("R,page,width,free,capacity,big", [
    (1, 16, 4, 3, 1, 0), (1, 64, 3, 2, 130, 100), (7, 48, 9, 100, 40, 20), (256, 64, 33, 300, 256 * 3, 0),
    (1023, 16, 12, 5000, 4000, 50), (1024, 32, 8, 100, 1024, 0), (1025, 16, 20, 4000, 20000, 120),
    (3000, 16, 40, 6000, 9000, 300), (2500, 128, 5, 0, 3000, 10)])
def test_page_plan_matches_sequential(D, R, page, width, free, capacity, big):
    case = plan_case(R, page, width, free, seed=R + page, capacity=capacity, big=big)
    got, want = run_plan(D, case), want_plan(case)
    wide = [c + n > width * page for c, n in zip(case[0].tolist(), case[1].tolist())]
    for k in want:
        assert got[k] == want[k], k
    if any(wide):
        expect_error(2)


@pytest.mark.parametrize("kw", [dict(alias=True), dict(cached_dtype=torch.int64), dict(stride=41)])
def test_page_plan_in_place_int64_and_strided(D, kw):
    case = plan_case(1500, 16, 40, 3000, seed=5, capacity=5000, big=30)
    got, want = run_plan(D, case, **kw), want_plan(case)
    for k in want:
        assert got[k] == want[k], k


def test_page_plan_no_requests_and_no_capacity(D):
    buf = D.page_plan_buffers(0, 4, DEV)
    for k in ("token_row", "positions", "slots"):
        buf[k].fill_(5)
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    D.page_plan(cached=e, new=e.clone(), block_table=torch.zeros(0, 3, dtype=torch.int32, device=DEV),
                free_ring=torch.zeros(4, dtype=torch.int32, device=DEV),
                ring_in=torch.tensor([2, 5], dtype=torch.int64, device=DEV), page_size=16, **buf)
    assert buf["token_row"].tolist() == [-1] * 4 and buf["ring_out"].tolist() == [2, 5] and buf["cu_new"].tolist() == [0]
    case = plan_case(5, 16, 4, 20, seed=3, capacity=0, finish=False)
    got, want = run_plan(D, case), want_plan(case)
    for k in want:
        assert got[k] == want[k], k


def test_page_plan_flags_impossible_input(D):
    # negative lengths, a request wider than its table row: not served, flagged, others unharmed
    case = plan_case(4, 16, 3, 20, seed=1, capacity=64, finish=False)
    cached, new = case[0], case[1]
    cached[:] = torch.tensor([5, -4, 40, 7])
    case[2][:] = torch.arange(12).view(4, 3)
    new[:] = torch.tensor([2, 1, 30, 1])
    got = run_plan(D, case)
    expect_error(2)
    assert got["counts"][3] == 2 and got["lens"][0] == 7 and got["lens"][3] == 8
    assert got["slots"][0] >= 0 and got["slots"][2 + 1] == -1
    # a ring that claims more pages than it holds frees none
    case = plan_case(3, 16, 3, 20, seed=2, capacity=64, finish=False)
    case = (*case[:4], (0, 10 ** 6), *case[5:])
    got = run_plan(D, case)
    expect_error(2)
    assert got["counts"][1] == 0


# ------------------------------------------------------------------ write / read
@pytest.mark.parametrize("n,page,scale", [(1, 16, 1.0), (5, 16, 1.0), (33, 48, 30.0), (257, 64, 1e-3), (1001, 128, 1.0)])
def test_latent4_write_and_read_bit_exact(D, n, page, scale):
    rows = rows_of(n, n, scale)
    pages = -(-n // page) + 3
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * page, generator=g)[:n]
    slots[::7] = -1
    cache = torch.randint(0, 256, (pages, page // 16 * 6400), generator=g, dtype=torch.uint8)
    want = cache.clone()
    S.write(rows, slots, want)
    got = cache.to(DEV)
    D.latent4_write(rows=rows.to(DEV), slots=slots.to(DEV), cache=got)
    assert torch.equal(got.cpu(), want)                  # other slots keep their bytes
    out = torch.full((n, 576), 7.0, dtype=torch.bfloat16, device=DEV)
    assert D.latent4_read(cache=got, slots=slots.to(DEV), out=out) is out
    expect = torch.where(slots[:, None] >= 0, S.values(rows), 0.0)
    assert torch.equal(out.cpu().double(), expect)


def test_latent4_edge_values_and_strides(D):
    # zeros, one huge element, saturation, scales on rounding ties, the smallest scales
    rows = rows_of(64, 9)
    rows[0] = 0
    rows[1, 5] = 3e4
    rows[2] = torch.linspace(-1e4, 1e4, 576).to(torch.bfloat16)
    rows[3] *= 1e-5
    rows[4] *= 1e-30
    for i in range(5, 40):                                # amax = 7 (2 m + 1) / 16: halfway scales
        rows[i, :512] = rows[i, :512].clamp(-0.5, 0.5)
        rows[i, ::32] = 7 * (2 * (i % 8 + 8) + 1) / 16
    wide = torch.zeros(64, 600, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:584] = rows.to(DEV)
    slots = torch.arange(64) + 16
    cache = torch.zeros(6, 6400, dtype=torch.uint8)
    want = cache.clone()
    S.write(rows, slots, want)
    got = cache.to(DEV)
    D.latent4_write(rows=wide[:, 8:584], slots=slots.to(DEV), cache=got)
    assert torch.equal(got.cpu(), want)
    out = torch.full((64, 600), 7.0, dtype=torch.bfloat16, device=DEV)
    D.latent4_read(cache=got, slots=slots.to(DEV), out=out[:, 16:592])
    assert torch.equal(out[:, 16:592].cpu().double(), S.values(rows))
    assert bool((out[:, :16] == 7).all() and (out[:, 592:] == 7).all())


def test_latent4_nonfinite_and_out_of_range(D):
    for bad, at in ((math.nan, 3), (math.inf, 100), (-math.inf, 511), (math.nan, 540)):
        rows = rows_of(3, 4)
        rows[1, at] = bad
        cache = torch.zeros(2, 6400, dtype=torch.uint8, device=DEV)
        slots = torch.tensor([1, 17, 31], device=DEV)
        D.latent4_write(rows=rows.to(DEV), slots=slots, cache=cache)
        expect_error(4)
        out = torch.empty(3, 576, dtype=torch.bfloat16, device=DEV)
        D.latent4_read(cache=cache, slots=slots, out=out)
        torch.testing.assert_close(out.cpu().double(), S.values(rows), rtol=0, atol=0, equal_nan=True)
    cache = torch.zeros(2, 6400, dtype=torch.uint8, device=DEV)
    rows = rows_of(2, 4).to(DEV)
    D.latent4_write(rows=rows, slots=torch.tensor([32, 10 ** 12], device=DEV), cache=cache)
    expect_error(2)
    assert not bool(cache.any())
    D.latent4_read(cache=cache, slots=torch.tensor([32, 5], device=DEV), out=rows)
    expect_error(2)
    assert not bool(rows.any())
    D.latent4_write(rows=rows[:0], slots=torch.zeros(0, dtype=torch.int64, device=DEV), cache=cache)


def test_mla_prep_q4_equals_prep_then_write(D):
    g = torch.Generator().manual_seed(3)
    B, L = 9, 70
    parts = torch.randn(3, B, 3648, generator=g).to(DEV)
    w = (1 + 0.2 * torch.randn(512, generator=g)).to(torch.bfloat16).to(DEV)
    ang = torch.rand(L, 32, generator=g) * 6
    cos, sin = torch.cos(ang).to(DEV), torch.sin(ang).to(DEV)
    pos = torch.tensor([0, 5, 69, 7, 7, 31, 2, 1, 16], device=DEV)
    slots = torch.tensor([3, 17, 40, -1, 0, 63, 16, 2, 33], device=DEV)
    for qkva in (parts, parts[0].to(torch.bfloat16)):
        ref = torch.zeros(B, L, 576, dtype=torch.bfloat16, device=DEV)
        pe, pe4 = (torch.zeros(B, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        no, no4 = (torch.zeros(B, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        D.mla_prep(qkva=qkva, kv_norm_w=w, eps=1e-6, cos=cos, sin=sin, positions=pos, cache=ref, q_pe_out=pe, q_nope_out=no)
        want = torch.zeros(4, 6400, dtype=torch.uint8, device=DEV)
        D.latent4_write(rows=ref[torch.arange(B), pos], slots=slots, cache=want)
        got = torch.zeros_like(want)
        D.mla_prep_q4(qkva=qkva, kv_norm_w=w, eps=1e-6, cos=cos, sin=sin, positions=pos, slots=slots, cache=got,
                      q_pe_out=pe4, q_nope_out=no4)
        assert torch.equal(got, want) and torch.equal(pe, pe4) and torch.equal(no, no4)
    # a padding row (position -1) writes nothing and is no error; a slot past the cache is
    before = got.clone()
    D.mla_prep_q4(qkva=parts, kv_norm_w=w, eps=1e-6, cos=cos, sin=sin, positions=torch.full_like(pos, -1), slots=slots,
                  cache=got, q_pe_out=pe4)
    assert torch.equal(got, before)
    D.mla_prep_q4(qkva=parts, kv_norm_w=w, eps=1e-6, cos=cos, sin=sin, positions=pos, slots=slots + 64, cache=got,
                  q_pe_out=pe4)
    expect_error(2)


# ------------------------------------------------------------------ attention
SCALE = 192 ** -0.5


class Pages:
    """Sequences of given lengths in shuffled pages of a cache whose unused bytes are garbage."""

    def __init__(self, lens, page, seed, spare=3, first_page=0, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.lens = page, lens
        held = [-(-n // page) for n in lens]
        total = sum(held) + spare
        order = (torch.randperm(total, generator=g) + first_page).tolist()
        width = max(max(held), 1) + 2
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        self.rows = [rows_of(n, seed + 1 + i, scale) for i, n in enumerate(lens)]
        blocks = page // 16
        cache = torch.randint(0, 256, (total, blocks * 6400), generator=g, dtype=torch.uint8)
        at = 0
        for i, n in enumerate(lens):
            pages = order[at:at + held[i]]
            at += held[i]
            self.table[i, :held[i]] = torch.tensor(pages, dtype=torch.int32)
            if n:
                slots = torch.tensor([(pages[t // page] - first_page) * page + t % page for t in range(n)])
                S.write(self.rows[i], slots, cache)
        self.cache = cache.to(DEV)

    def values(self, i, n):
        v = S.values(self.rows[i][:n])
        return v[:, :512], v[:, 512:]


def queries(rows, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(rows, 16, 512, generator=g) * scale).to(torch.bfloat16),
            (torch.randn(rows, 16, 64, generator=g) * scale).to(torch.bfloat16))


def check_attention(D, pg, q, positions, seq_rows=None, scale=SCALE, cache=None, rows=None):
    q_abs, q_pe = q
    n = q_abs.shape[0]
    out = torch.full((n, 16, 512), math.nan, dtype=torch.bfloat16, device=DEV)
    args = dict(q_abs=q_abs.to(DEV), q_pe=q_pe.to(DEV), cache=pg.cache if cache is None else cache,
                block_table=pg.table.to(DEV), positions=torch.tensor(positions, device=DEV), page_size=pg.page,
                softmax_scale=scale, seq_rows=None if seq_rows is None else torch.tensor(seq_rows, dtype=torch.int32, device=DEV))
    ws = D.mla_q4_workspace(n, DEV)
    assert D.mla_decode_q4(**args, o_lat=out, **ws) is out
    first = out.clone()
    out.fill_(math.nan)
    D.mla_decode_q4(**args, o_lat=out, **ws)
    assert torch.equal(first, out)                       # same bits again, nothing left behind
    got = out.cpu().double()
    for r in (range(n) if rows is None else rows):
        s = r if seq_rows is None else seq_rows[r]
        m = 0 if s < 0 else positions[r] + 1
        lat, rope = pg.values(s, m) if m > 0 else (torch.zeros(0, 512).double(), torch.zeros(0, 64).double())
        want, mag, terms = S.attention(q_abs[r].double(), q_pe[r].double(), lat, rope, scale)
        d = 576 * 2 ** -24 * terms
        bad = (got[r] - want).abs() - (2 ** -7 + 2 * d) * mag - 1e-30
        assert float(bad.max()) <= 0, (r, m, float((got[r] - want).abs().max()))
        if m == 0:
            assert not bool(got[r].any())
    return out


@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_attention_lengths_around_blocks_tiles_and_pages(D, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 47, 48, 49, 63, 64, 65, 96, 127, 128, 129, 200, 255, 257, 300]
    pg = Pages(lens, page, seed=page)
    check_attention(D, pg, queries(len(lens), 1), [n - 1 for n in lens])


def test_attention_empty_rows_and_shared_sequences(D):
    lens = [40, 0, 130, 1]
    pg = Pages(lens, 32, seed=5)
    # several rows per sequence at different positions, rows without a sequence, rows of position -1
    seq = [2, 2, 2, -1, 0, 1, 3, 0, 2, -5]
    pos = [129, 64, 0, 10, -1, -1, 0, 39, 100, -1]
    check_attention(D, pg, queries(len(seq), 2), pos, seq)
    check_attention(D, pg, queries(1, 2), [-1], [1])     # nothing to do at all


@pytest.mark.parametrize("lens", [[3000], [5000, 1], [1] * 300, [700] * 40 + [9000]])
def test_attention_long_rows_and_many_rows(D, lens):
    pg = Pages(lens, 64, seed=len(lens))
    n = len(lens)
    rows = sorted({0, 1, 2, n // 2, n - 2, n - 1} & set(range(n)))
    check_attention(D, pg, queries(n, 7), [v - 1 for v in lens], rows=rows)


@pytest.mark.parametrize("qs,scale", [(1e-6, SCALE), (300.0, 1e-4), (1.0, 5.0), (1.0, 0.0), (2e20, 1e-22), (1e-25, 1e22)])
def test_attention_query_and_score_ranges(D, qs, scale):
    # tiny and huge queries, a softmax that is one-hot, one that is flat
    pg = Pages([5, 70, 333], 16, seed=11)
    check_attention(D, pg, queries(3, 3, qs), [4, 69, 332], scale=scale)


def test_attention_values_of_saturated_and_zero_groups(D):
    for s in (1e3, 1e-4, 0.0):
        pg = Pages([90, 17], 48, seed=12, scale=s)
        check_attention(D, pg, queries(2, 4, 1e-3), [89, 16])


def test_attention_pages_past_four_gigabytes(D):
    pg = Pages([50, 20], 64, seed=13, first_page=180000)
    page_bytes = 4 * 6400
    cache = torch.empty((180000 + pg.cache.shape[0], page_bytes), dtype=torch.uint8, device=DEV)
    cache[180000:] = pg.cache
    check_attention(D, pg, queries(2, 5), [49, 19], cache=cache)


def test_attention_on_another_stream_and_in_a_graph(D):
    pg = Pages([100, 300, 7], 64, seed=14)
    q_abs, q_pe = (t.to(DEV) for t in queries(3, 6))
    pos = torch.tensor([99, 299, 6], device=DEV)
    table = pg.table.to(DEV)
    want = check_attention(D, pg, queries(3, 6), [99, 299, 6])
    ws = D.mla_q4_workspace(3, DEV)
    out = torch.zeros_like(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def call():
        D.mla_decode_q4(q_abs=q_abs, q_pe=q_pe, cache=pg.cache, block_table=table, positions=pos, page_size=64,
                        softmax_scale=SCALE, o_lat=out, **ws)
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_attention_flags_pages_and_rows_out_of_range(D):
    pg = Pages([40, 40, 40], 16, seed=15)
    pg.table[1, 1] = 10 ** 6                              # a page that the cache does not have
    q_abs, q_pe = (t.to(DEV) for t in queries(3, 6))
    out = torch.zeros(3, 16, 512, dtype=torch.bfloat16, device=DEV)

    def call(positions, seq_rows):
        D.mla_decode_q4(q_abs=q_abs, q_pe=q_pe, cache=pg.cache, block_table=pg.table.to(DEV),
                        positions=torch.tensor(positions, device=DEV), page_size=16, softmax_scale=SCALE, o_lat=out,
                        seq_rows=torch.tensor(seq_rows, dtype=torch.int32, device=DEV), **D.mla_q4_workspace(3, DEV))
        torch.cuda.synchronize()
    call([39, 39, 39], [0, 1, 2])
    expect_error(2)
    call([39, 39, 39], [0, 7, 2])                         # a table row that does not exist
    expect_error(2)
    call([39, 10 ** 9, 39], [0, 1, 2])                    # a length beyond the table
    expect_error(2)
    check_attention(D, pg, queries(3, 6), [39, 39, 39], [0, 2, 2])   # and fine again


# ------------------------------------------------------------------ adapters
def lora_case(T, n_ad, rank, K, N, seed, none=0.2, ranks=None):
    g = torch.Generator().manual_seed(seed)

    def bf(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)
    c = {"x": bf(T, K), "w": bf(N, K, std=0.02), "a": bf(n_ad, rank, K, std=K ** -0.5), "b": bf(n_ad, N, rank, std=0.05),
         "ids": torch.randint(0, n_ad, (T,), generator=g, dtype=torch.int32),
         "ranks": torch.randint(0, rank + 1, (n_ad,), generator=g, dtype=torch.int32),
         "scales": torch.rand(n_ad, generator=g) * 3 - 1}
    c["ids"][torch.rand(T, generator=g) < none] = -1
    c["ranks"][0] = rank
    if ranks:
        c["ranks"] = torch.tensor(ranks, dtype=torch.int32)
    # rows past an adapter's rank are not part of it, whatever they hold
    for i, r in enumerate(c["ranks"].tolist()):
        c["a"][i, r:] = math.nan
        c["b"][i, :, r:] = math.nan
    return c


def check_lora(got, c, w=True, out_bits=8):
    y, low, mag = S.lora(c["x"], c["w"] if w else None, c["a"], c["b"], c["ids"].tolist(), c["ranks"], c["scales"])
    tol = 2.0 ** -out_bits * y.abs() + 2 ** -8 * low + c["x"].shape[1] * 2 ** -23 * mag + 1e-30
    bad = (got.cpu().double() - y).abs() - tol
    assert not bool(got.isnan().any()) and float(bad.max()) <= 0, float(bad.max())


@pytest.mark.parametrize("T,n_ad,rank,K,N", [
    (1, 1, 8, 64, 8), (1, 5, 16, 2048, 3648), (2, 3, 8, 128, 72), (7, 2, 64, 2048, 2048), (8, 9, 24, 192, 136),
    (9, 4, 16, 2048, 3648), (33, 33, 40, 256, 520), (100, 1, 128, 320, 264), (257, 7, 64, 2048, 1000),
    (300, 33, 16, 128, 96), (1030, 64, 128, 128, 136), (2049, 1, 24, 64, 1288),
    (700, 20, 32, 2048, 512), (129, 3, 56, 10944, 128), (1100, 2, 8, 64, 40)])
def test_lora_linear(D, T, n_ad, rank, K, N):
    c = lora_case(T, n_ad, rank, K, N, seed=T + N)
    d = {k: v.to(DEV) for k, v in c.items()}
    y = torch.full((T, N), math.nan, dtype=torch.bfloat16, device=DEV)
    ws = D.lora_workspace(T, N, K, rank, DEV)
    assert D.lora_linear(**d, y=y, **ws) is y
    check_lora(y, c)
    first = y.clone()
    D.lora_linear(**d, y=y, **ws)
    assert torch.equal(y, first)


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_lora_alone_strided_and_by_request(D, T):
    c = lora_case(T, 4, 16, 256, 200, seed=T)
    ids = c["ids"].clone()
    # ids per request, tokens in shuffled requests, padding rows at the end
    g = torch.Generator().manual_seed(T)
    req = torch.randperm(T, generator=g)
    token_row = req.to(torch.int32)
    token_row[T - T // 4:] = -1
    by_req = torch.empty_like(ids)
    by_req[req] = ids
    c["ids"] = torch.where(token_row < 0, torch.tensor(-1, dtype=torch.int32), ids)
    x = torch.full((T, 304), math.nan, dtype=torch.bfloat16, device=DEV)
    x[:, 8:264] = c["x"].to(DEV)
    y = torch.full((T, 208), 5.0, device=DEV)
    low = torch.empty(T * 16, device=DEV)
    D.lora(x=x[:, 8:264], a=c["a"].to(DEV), b=c["b"].to(DEV), ids=by_req.to(DEV), token_row=token_row.to(DEV),
           ranks=c["ranks"].to(DEV), scales=c["scales"].to(DEV), y=y[:, :200], low=low, order=torch.empty(3 * T, dtype=torch.int32, device=DEV))
    check_lora(y[:, :200], c, w=False, out_bits=20)
    assert bool((y[:, 200:] == 5).all())
    assert not bool(y[:, :200][c["ids"].to(DEV) < 0].any())


def test_lora_rows_without_adapter_keep_the_projection(D):
    c = lora_case(50, 2, 8, 512, 96, seed=1, none=1.1)
    d = {k: v.to(DEV) for k, v in c.items()}
    y = torch.empty(50, 96, dtype=torch.bfloat16, device=DEV)
    D.lora_linear(**d, y=y, **D.lora_workspace(50, 96, 512, 8, DEV))
    check_lora(y, c)


@pytest.mark.parametrize("T,rank,N", [(1, 8, 64), (6, 16, 72), (16, 40, 200), (100, 16, 264), (300, 24, 520), (520, 64, 104)])
def test_lora_infinities_stay_with_their_adapter(D, T, rank, N):
    c = lora_case(T, 3, rank, 256, N, seed=T, ranks=[rank, rank - 1, rank - 5])
    c["ids"][0] = 1

    def run():
        y = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
        D.lora_linear(**{k: v.to(DEV) for k, v in c.items()}, y=y, **D.lora_workspace(T, N, 256, rank, DEV))
        return y.cpu()
    clean = run()
    c["b"][1, 3, 2], c["b"][1, N - 1, 0], c["b"][1, 17, rank - 2] = math.inf, math.nan, -math.inf
    got = run()
    own = c["ids"] == 1
    assert torch.equal(got[~own], clean[~own])            # other adapters' tokens do not see them
    keep = [n for n in range(N) if n not in (3, 17, N - 1)]
    assert torch.equal(got[own][:, keep], clean[own][:, keep])
    want, _, _ = S.lora(c["x"], c["w"], c["a"], c["b"], c["ids"].tolist(), c["ranks"], c["scales"])
    assert torch.equal(got[own][:, [3, 17]].double(), want[own][:, [3, 17]])
    assert bool(got[own][:, N - 1].isnan().all())


@pytest.mark.parametrize("T,rank", [(300, 16), (777, 40)])
def test_lora_long_runs_strided_by_request_in_a_graph(D, T, rank):
    K, N = 192, 328
    c = lora_case(T, 5, rank, K, N, seed=T)
    g = torch.Generator().manual_seed(T)
    req = torch.randperm(T, generator=g)
    token_row = req.to(torch.int32)
    token_row[T - 20:] = -1                               # padding rows: the projection alone
    by_req = torch.empty_like(c["ids"])
    by_req[req] = c["ids"]
    c["ids"] = torch.where(token_row < 0, torch.tensor(-1, dtype=torch.int32), c["ids"])
    x = torch.full((T, K + 40), math.nan, dtype=torch.bfloat16, device=DEV)
    x[:, 8:8 + K] = c["x"].to(DEV)
    w = torch.full((N, K + 16), math.nan, dtype=torch.bfloat16, device=DEV)
    w[:, :K] = c["w"].to(DEV)
    y = torch.full((T, N + 24), 5.0, dtype=torch.bfloat16, device=DEV)
    d = {k: c[k].to(DEV) for k in ("a", "b", "ranks", "scales")}
    ids, token_row = by_req.to(DEV), token_row.to(DEV)
    ws = D.lora_workspace(T, N, K, rank, DEV)
    ws["xs"].fill_(math.nan)                              # work buffers may hold anything
    ws["lists"].fill_(-7)

    def run():
        D.lora_linear(x=x[:, 8:8 + K], w=w[:, :K], ids=ids, token_row=token_row, y=y[:, :N], **d, **ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    s.synchronize()
    check_lora(y[:, :N], c)
    first = y.clone()
    assert bool((y[:, N:] == 5).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    y[:, :N] = 0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)


def test_lora_refuses_short_gemm_buffers(D):
    c = lora_case(300, 2, 16, 64, 64, seed=3)
    d = {k: v.to(DEV) for k, v in c.items()}
    y = torch.empty(300, 64, dtype=torch.bfloat16, device=DEV)
    ws = D.lora_workspace(300, 64, 64, 16, DEV)
    for name in ("xs", "lists"):
        with pytest.raises(ValueError):
            D.lora_linear(**d, y=y, **dict(ws, **{name: ws[name].view(-1)[:-1]}))
    with pytest.raises(ValueError):                       # not on a 16-byte boundary
        D.lora_linear(**d, y=y, **dict(ws, xs=torch.empty(ws["xs"].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:]))


def test_lora_flags_ids_out_of_range(D):
    c = lora_case(20, 2, 8, 64, 16, seed=2, none=0)
    good = c["ids"].clone()
    c["ids"][3] = 2
    d = {k: v.to(DEV) for k, v in c.items()}
    y = torch.empty(20, 16, dtype=torch.bfloat16, device=DEV)
    ws = D.lora_workspace(20, 16, 64, 8, DEV)
    D.lora_linear(**d, y=y, **ws)
    torch.cuda.synchronize()
    expect_error(2)
    c["ids"][3] = -1                                      # such a row has no adapter
    check_lora(y, c)
    c["ids"] = good
    d["ids"] = good.to(DEV)
    D.lora_linear(**d, y=y, **ws)
    check_lora(y, c)
