"""What the serving operators keep of their inputs' precision, with bounds for each path of the adapters and
rows of attention that one token decides."""
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


# ------------------------------------------------------------------ adapters
# Bounds, from the roundings of each path: low is an fp32 sum; up to 16 tokens of lora_linear it is used as it is,
# elsewhere as the sum of two bf16 numbers, each within 2^-8 of what it stands for: 2^-16 of low is lost.  The
# fp32 sums of the K products of W x and of low are off by at most (K + 512) 2^-24 of the sum of their
# magnitudes, the sum over the ranks (two products each, truncated) by (2 rank + 64) 2^-23, and the result's own
# rounding is 2^-8 (bf16) or 2^-24 (fp32) of it.
def lora_tol(c, y, low, mag, split, f32):
    k, rank = c["x"].shape[1] + 512, c["a"].shape[1]
    return ((2.0 ** -24 if f32 else 2.0 ** -8) * y.abs() + (2.0 ** -16 if split else 0.0) * low * (1 + 2.0 ** -7) +
            (2 * rank + 64) * 2.0 ** -23 * low + k * 2.0 ** -24 * mag + 1e-30)


def lora_case(T, n_ad, rank, K, N, seed, cancel=False):
    g = torch.Generator().manual_seed(seed)

    def bf(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)
    c = {"x": bf(T, K), "w": bf(N, K, std=0.02), "a": bf(n_ad, rank, K, std=K ** -0.5), "b": bf(n_ad, N, rank, std=0.5),
         "ids": torch.randint(-1, n_ad, (T,), generator=g, dtype=torch.int32),
         "ranks": torch.randint(max(2, rank - 7), rank + 1, (n_ad,), generator=g, dtype=torch.int32),
         "scales": torch.rand(n_ad, generator=g) + 0.5}
    if cancel:
        # ranks 0 and 1 cancel, 48 low_0 - 64 (3 / 4 low_0), and are far larger than what is left; x in 16ths up to 4 and
        # powers of two in A make both sums exact in fp32
        c["x"] = (torch.randn(T, K, generator=g) * 16).round().clamp(-64, 64).div(16).to(torch.bfloat16)
        e = torch.randint(0, 2, (n_ad, K), generator=g) - round(math.log2(K) / 2)
        c["a"][:, 0] = (torch.exp2(e.float()) * (torch.randint(0, 2, (n_ad, K), generator=g) * 2 - 1)).to(torch.bfloat16)
        c["a"][:, 1] = 0.75 * c["a"][:, 0]
        c["b"] *= 0.01
        c["b"][:, :, 0] = 48.0
        c["b"][:, :, 1] = -64.0
        c["w"] *= 0.05
    for i, r in enumerate(c["ranks"].tolist()):
        c["a"][i, r:] = math.nan
        c["b"][i, :, r:] = math.nan
    return c


def lora_want(c, w=True, cancel=False):
    """(y, sum |low B|, the magnitudes of the sums over k that are not exact)."""
    ids = c["ids"].tolist()
    y, low, mag = S.lora(c["x"], c["w"] if w else None, c["a"], c["b"], ids, c["ranks"], c["scales"])
    if cancel:
        b = c["b"].clone()
        b[:, :, :2] = 0
        mag = S.lora(c["x"], c["w"] if w else None, c["a"], b, ids, c["ranks"], c["scales"])[2]
    return y, low, mag


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("T,n_ad,rank,K,N", [
    (1, 2, 8, 2048, 256), (5, 3, 48, 256, 72), (8, 2, 128, 192, 136), (16, 5, 96, 320, 200), (13, 4, 64, 1024, 264),
    (3, 2, 16, 72, 40), (16, 3, 72, 584, 48), (17, 3, 16, 256, 200), (64, 20, 40, 2048, 264), (200, 9, 64, 512, 328),
    (257, 3, 16, 2048, 264), (400, 5, 40, 256, 520), (700, 30, 128, 192, 136), (300, 40, 24, 128, 72),
    (1030, 8, 128, 512, 264), (900, 12, 128, 2048, 136)])
def test_lora_linear_keeps_the_adapters_precision(D, T, n_ad, rank, K, N, cancel, f32):
    c = lora_case(T, n_ad, rank, K, N, seed=T + rank, cancel=cancel)
    y = torch.full((T, N), math.nan, dtype=torch.float32 if f32 else torch.bfloat16, device=DEV)
    D.lora_linear(**{k: v.to(DEV) for k, v in c.items()}, y=y, **D.lora_workspace(T, N, K, rank, DEV))
    want, low, mag = lora_want(c, cancel=cancel)
    bad = (y.cpu().double() - want).abs() / lora_tol(c, want, low, mag, split=T > 16, f32=f32)
    assert not bool(y.isnan().any()) and float(bad.max()) <= 1, float(bad.max())


@pytest.mark.parametrize("T,n_ad,rank,K,N", [(1, 2, 16, 72, 40), (9, 3, 128, 1096, 136), (40, 7, 56, 264, 328), (600, 12, 32, 520, 200)])
def test_lora_alone_keeps_precision_at_any_k(D, T, n_ad, rank, K, N):
    c = lora_case(T, n_ad, rank, K, N, seed=K)
    g = torch.Generator().manual_seed(1)
    base = torch.randn(3, T, N, generator=g)
    y = torch.empty(T, N, device=DEV)
    ws = D.lora_workspace(T, N, K, rank, DEV)
    D.lora(**{k: v.to(DEV) for k, v in c.items() if k != "w"}, y=y, base=base.to(DEV), low=ws["low"], order=ws["order"])
    want, low, mag = lora_want(c, w=False)
    want, mag = want + base.double().sum(0), mag + base.double().abs().sum(0)
    bad = (y.cpu().double() - want).abs() / lora_tol(c, want, low, mag, split=True, f32=True)
    assert float(bad.max()) <= 1, float(bad.max())


@pytest.mark.parametrize("T", [6, 40, 300])
def test_lora_infinities_on_both_sides(D, T):
    """An infinite low-rank activation that meets an infinity of B is an infinity (or, of opposite
    signs, a NaN), as in 64 bits, whatever the number of tokens."""
    K, N, rank = 256, 72, 24
    c = lora_case(T, 2, rank, K, N, seed=T)
    c["ranks"][:] = rank
    g = torch.Generator().manual_seed(7)
    c["a"] = (torch.randn(2, rank, K, generator=g) * K ** -0.5).to(torch.bfloat16)
    c["b"] = (torch.rand(2, N, rank, generator=g) + 0.25).to(torch.bfloat16)       # no zeros
    c["ids"][:] = torch.arange(T) % 3 - 1
    c["x"][:, 0] = 1.0
    c["a"][1, 3, 0] = math.inf                           # low[:, 3] of every token of adapter 1
    c["b"][1, 5, 3], c["b"][1, 9, 3], c["b"][1, 11, 6] = math.inf, -math.inf, math.inf
    c["b"][1, 13, 3] = -0.5
    y = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    D.lora_linear(**{k: v.to(DEV) for k, v in c.items()}, y=y, **D.lora_workspace(T, N, K, rank, DEV))
    want, low, mag = lora_want(c)
    y = y.cpu().double()
    own = c["ids"] == 1
    sane = want.isfinite()
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y[~sane & ~want.isnan()], want[~sane & ~want.isnan()])
    assert bool((~sane)[own].any()) and bool(sane[~own].all())
    tol = lora_tol(c, want, low, mag, split=T > 16, f32=False)
    assert float(((y - want).abs() / tol)[sane].max()) <= 1


# ------------------------------------------------------------------ attention
SCALE = 192 ** -0.5


class Pages:
    """Sequences of given lengths in shuffled pages (values of few distinct rows: quick to make)."""

    def __init__(self, D, lens, page, seed):
        g = torch.Generator().manual_seed(seed)
        self.page, self.lens = page, lens
        held = [-(-n // page) for n in lens]
        order = torch.randperm(sum(held) + 3, generator=g)
        self.table = torch.full((len(lens), max(held) + 2), -1, dtype=torch.int32)
        self.cache = torch.randint(0, 256, (sum(held) + 3, page // 16 * 6400), generator=g, dtype=torch.uint8).to(DEV)
        self.rows, at = [], 0
        for i, n in enumerate(lens):
            pages = order[at:at + held[i]]
            at += held[i]
            self.table[i, :held[i]] = pages.to(torch.int32)
            rows = torch.randn(n, 576, generator=g).to(torch.bfloat16)
            t = torch.arange(n)
            D.latent4_write(rows=rows.to(DEV), slots=(pages[t // page] * page + t % page).to(DEV), cache=self.cache)
            self.rows.append(S.values(rows))

    def run(self, D, q_abs, q_pe, positions, seq_rows=None, scale=SCALE, table=None):
        n = q_abs.shape[0]
        out = torch.full((n, 16, 512), math.nan, dtype=torch.bfloat16, device=DEV)
        D.mla_decode_q4(q_abs=q_abs.to(DEV), q_pe=q_pe.to(DEV), cache=self.cache,
                        block_table=self.table.to(DEV) if table is None else table,
                        positions=torch.tensor(positions, device=DEV), page_size=self.page, softmax_scale=scale, o_lat=out,
                        seq_rows=None if seq_rows is None else torch.tensor(seq_rows, dtype=torch.int32, device=DEV),
                        **D.mla_q4_workspace(n, DEV))
        return out.cpu().double()


@pytest.mark.parametrize("n,page", [(1, 16), (70, 16), (513, 48), (3000, 64), (9001, 64)])
def test_attention_counts_every_token_once(D, n, page):
    """Head h sees eight tokens alone (at block, tile and page edges, the first and the last among them), all with the same
    score: its result is the mean of their rows.  A token lost or counted twice moves it by a tenth of a row."""
    pg = Pages(D, [n], page, seed=n)
    g = torch.Generator().manual_seed(n + 1)
    edges = torch.tensor(sorted({t for b in range(0, n, 16) for t in (b, b + 15) if t < n} | {n - 1}))
    q_pe = torch.zeros(1, 16, 64)
    q_pe[0, torch.arange(16), torch.arange(16)] = 16.0
    for batch in range(3):
        rows = pg.rows[0].to(torch.bfloat16)              # (exact: quantised values are bf16 numbers)
        rows[:, 512:] = 0
        groups = []
        for h in range(16):
            pick = edges[torch.randperm(len(edges), generator=g)[:8]]
            if h < 4:
                pick[0] = n - 1 if h % 2 else 0
            groups.append(pick.unique())
            rows[groups[-1], 512 + h] = 16.0              # score 256 against 0
        t = torch.arange(n)
        slots = pg.table[0].long()[t // page] * page + t % page
        D.latent4_write(rows=rows.to(DEV), slots=slots.to(DEV), cache=pg.cache)
        val = S.values(rows)[:, :512]
        got = pg.run(D, torch.zeros(1, 16, 512, dtype=torch.bfloat16), q_pe.to(torch.bfloat16), [n - 1], scale=1.0)[0]
        for h, grp in enumerate(groups):
            want, mag = val[grp].mean(0), val[grp].abs().mean(0)
            # the result's bf16 rounding; sums of at most 8 products of 8-bit numbers, in fp32
            assert float(((got[h] - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -18 * mag - 1e-30).max()) <= 0, (batch, h)


def test_attention_divides_by_the_probabilities_that_it_multiplies(D):
    """Every token holds the same latent row, so the result is that row, a bf16 number, whatever the probabilities are
    rounded to, if their sum is that of the rounded ones.  Token 130 has 128.05 .. 128.95 times the probability of token 0,
    in a later tile (where the maximum is not taken anew: it would round by up to 2^-8); the others have none."""
    n, R = 144, 2000
    pg = Pages(D, [n], 16, seed=1)
    rows = torch.randn(1, 576, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).repeat(n, 1)
    rows[:, 512:] = 0
    rows[130, 512], rows[130, 513] = 1, 1
    rows[:, 514] = 1
    rows[0, 514] = rows[130, 514] = 0
    t = torch.arange(n)
    D.latent4_write(rows=rows.to(DEV), slots=(pg.table[0].long()[t // 16] * 16 + t % 16).to(DEV), cache=pg.cache)
    q_pe = torch.zeros(16, 64)
    q_pe[:, 0] = 7.0
    q_pe[:, 1] = torch.log2(1 + torch.linspace(0.05, 0.95, 16) / 128)
    q_pe[:, 2] = -1000.0
    got = pg.run(D, torch.zeros(R, 16, 512, dtype=torch.bfloat16), q_pe.to(torch.bfloat16).expand(R, 16, 64).contiguous(),
                 [n - 1] * R, [0] * R, scale=math.log(2))
    want = S.values(rows[:1])[:, :512].expand(R, 16, 512)
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("R", [639, 640, 641, 1290])
def test_attention_of_many_rows(D, R):
    """Prompt rows: more query rows than the launch has threads, several sequences, tables with wide rows."""
    lens = [211, 90, 330, 17]
    pg = Pages(D, lens, 32, seed=R)
    g = torch.Generator().manual_seed(R)
    seq = torch.randint(-1, len(lens), (R,), generator=g).tolist()
    pos = [int(torch.randint(0, lens[s], (1,), generator=g)) if s >= 0 else 3 for s in seq]
    q_abs = torch.randn(R, 16, 512, generator=g).to(torch.bfloat16)
    q_pe = torch.randn(R, 16, 64, generator=g).to(torch.bfloat16)
    wide = torch.full((len(lens), pg.table.shape[1] + 5), 10 ** 6, dtype=torch.int32)
    wide[:, :pg.table.shape[1]] = pg.table
    got = pg.run(D, q_abs, q_pe, pos, seq, table=wide.to(DEV)[:, :pg.table.shape[1]])
    for r in sorted({0, 1, R // 2, 638, R - 2, R - 1} | set(range(5, R, 37))):
        m = 0 if seq[r] < 0 else pos[r] + 1
        v = pg.rows[seq[r]][:m] if m else torch.zeros(0, 576).double()
        want, mag, terms = S.attention(q_abs[r].double(), q_pe[r].double(), v[:, :512], v[:, 512:], SCALE)
        # the stored probabilities and the result in bf16, scores off by d in the exponent
        d = 576 * 2.0 ** -24 * terms
        assert float(((got[r] - want).abs() - (2.0 ** -7 + 2 * d) * mag - 1e-30).max()) <= 0, r
        if m == 0:
            assert not bool(got[r].any())
