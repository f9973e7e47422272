"""Cases of the paged 4-bit serving operators: what is timed, with plain forms and 64-bit values.

Four operators of a decode step that serves many requests from one paged latent cache held
in 4 bits, each request with its own low-rank adapter:

  plan   page tables, token slots and positions of a step, from the requests' lengths
  write  latent rows quantised into their slots (and read back as the values they stand for)
  attn   latent attention over the 4-bit pages
  lora   a shared projection plus each row's own low-rank adapter

`run` computes them with elementary torch operations in fp32 where `own` is false, and
through the `dsv2.ops` entry points where it is true.

The 4-bit cache is an array of 16-token blocks of 6400 bytes (a page is page_size / 16 of
them; slot = page * page_size + offset, block = slot // 16, p = slot % 16):

  [0, 4096)     token p at 256 p: the 16 groups of 32 latent dims, 16 bytes each, group c at
                place c ^ f(p), f(p) = 2 (p & 1) + 4 ((p >> 1 ^ p >> 2) & 1); word w of a group
                holds dims 8 w .. 8 w + 7, dim 8 w + 2 i in its nibble i and 8 w + 2 i + 1 in
                nibble 4 + i, as value / scale + 8
  [4096, 4352)  scale codes, group c of token p at 4096 + 16 c + 4 (p & 3) + (p >> 2): the
                scale is the positive fp16 number whose bits are code << 7 (3 mantissa bits)
  [4352, 6400)  token p at 4352 + 128 p: the 64 roped dims in bf16, 8 chunks of 8 dims, chunk j
                at place j ^ (p & 4)
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
HEADS, LATENT, ROPE, ROW = 16, 512, 64, 576
BLOCK_TOKENS, BLOCK_BYTES = 16, 6400
MAX_CODE = 167                      # scale 60, the largest whose products with the nibbles stay in fp16
SOFTMAX_SCALE = 192 ** -0.5


def _ops():
    root = str(Path("flash-deepseek-v2-lite_b200").resolve())
    if root not in sys.path:
        sys.path.insert(0, root)
    from dsv2 import ops
    return ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of 256 running requests: one token each, few of them open a page
        {"name": "plan_decode_256", "op": "plan", "requests": 256, "tokens": 0, "page": 64, "max_len": 2048},
        # a mixed step: decoding requests, chunks of prompts up to 4096 tokens, finished requests, 16-token pages
        {"name": "plan_mixed_1500", "op": "plan", "requests": 1500, "tokens": 16381, "page": 16, "max_len": 8192},
        # the new rows of one decode step of 32 requests, some of them padding
        {"name": "write_decode_32", "op": "write", "rows": 32, "page": 64, "pad": 8},
        # the rows of several prompts' chunks (ragged, odd)
        {"name": "write_prefill_16381", "op": "write", "rows": 16381, "page": 64, "pad": 50},
        # one request at a 512-token context: latency
        {"name": "attn_b1_512", "op": "attn", "seqs": 1, "queries": 1, "lo": 512, "hi": 512, "page": 64, "empty": 0},
        # 32 requests at 512 tokens
        {"name": "attn_b32_512", "op": "attn", "seqs": 32, "queries": 1, "lo": 500, "hi": 530, "page": 64, "empty": 0},
        # 256 ragged requests, some rows of the batch unused, small pages
        {"name": "attn_b256_ragged", "op": "attn", "seqs": 256, "queries": 1, "lo": 128, "hi": 1024, "page": 16, "empty": 17},
        # long contexts: the cache reads are all there is
        {"name": "attn_b64_8192", "op": "attn", "seqs": 64, "queries": 1, "lo": 8192, "hi": 8192, "page": 64, "empty": 0},
        # three draft tokens a request checked at once, one long request among short ones
        {"name": "attn_b9_q3_ragged", "op": "attn", "seqs": 9, "queries": 3, "lo": 3, "hi": 12001, "page": 48, "empty": 0},
        # one token through the query + latent projection with its request's adapter
        {"name": "lora_1", "op": "lora", "rows": 1, "adapters": 4, "rank": 16, "k": 2048, "n": 3648},
        # 200 decoding requests, 40 adapters of mixed ranks
        {"name": "lora_200_mixed", "op": "lora", "rows": 200, "adapters": 40, "rank": 64, "k": 2048, "n": 3648},
        # a prompt chunk through the same projection, few adapters
        {"name": "lora_4001", "op": "lora", "rows": 4001, "adapters": 6, "rank": 32, "k": 2048, "n": 3648},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attn", "attn", "lora", "lora"])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 4000), "tokens": rng.choice([0, _log(rng, 1, 16381)]),
                "page": rng.choice([16, 32, 48, 64, 128]), "max_len": _log(rng, 256, 8192)}
    if op == "write":
        return {"op": op, "rows": _log(rng, 1, 16381), "page": rng.choice([16, 48, 64, 128]), "pad": rng.choice([0, 3, 50])}
    if op == "attn":
        queries = rng.choice([1, 1, 1, 2, 5])
        hi = _log(rng, max(8, queries), 16000)
        seqs = _log(rng, 1, min(300, max(1, 400000 // (hi * queries))))
        return {"op": op, "seqs": seqs, "queries": queries, "lo": max(queries, rng.randrange(1, hi + 1)), "hi": hi,
                "page": rng.choice([16, 32, 48, 64, 128]), "empty": rng.choice([0, 0, 5])}
    k, n = rng.choice([(2048, 3648), (2048, 2048), (10944, 2048)])
    return {"op": op, "rows": _log(rng, 1, 1200 if k > 4096 else 3800), "adapters": _log(rng, 1, 60),
            "rank": rng.choice([8, 16, 32, 48, 64]), "k": k, "n": n}


def _lens(case):
    """Lengths of the sequences, shortest to longest; every `empty`-th has none."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    out = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    return [0 if case["empty"] and i % case["empty"] == 1 else v for i, v in enumerate(out)]


def _ranks(case):
    return [max(1, case["rank"] - 5 * (a % 4)) for a in range(case["adapters"])]


def work(case):
    op = case["op"]
    if op == "plan":
        r, t = case["requests"], max(case["tokens"], case["requests"])
        return {"bytes": float(r * (4 + 4 + 4 + 4) + t * (4 + 8 + 8)), "flops": float(4 * r + 6 * t)}
    if op == "write":
        t = case["rows"]
        return {"bytes": float(t * (1152 + 8 + 400) + t * (400 + 8 + 1152)), "flops": float(t * LATENT * 6)}
    if op == "attn":
        tokens, rows = sum(_lens(case)), case["seqs"] * case["queries"]
        return {"bytes": float(tokens * 400 + rows * HEADS * (ROW + LATENT) * 2),
                "flops": float(tokens * case["queries"] * HEADS * 2 * (ROW + LATENT))}
    t, k, n = case["rows"], case["k"], case["n"]
    ranks = _ranks(case)
    used = sum(ranks[:min(len(ranks), t)])
    mean = sum(ranks) / len(ranks)
    return {"bytes": float(2 * (t * k + k * n + t * n + used * (k + n))), "flops": float(2 * t * k * n + 2 * t * mean * (k + n))}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _latent_rows(n, g):
    """Latent rows as the cache gets them: the norm's output times its weights, and roped keys."""
    x = torch.randn(n, ROW, generator=g, device=DEV)
    w = 0.5 + torch.rand(LATENT, generator=g, device=DEV)
    c = x[:, :LATENT]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6) * w
    return torch.cat([c, x[:, LATENT:]], 1).to(torch.bfloat16)


def _prepare_plan(case, g):
    r, page, max_len = case["requests"], case["page"], case["max_len"]
    cached = torch.randint(0, max_len - 1, (r,), generator=g, device=DEV, dtype=torch.int32)
    new = torch.ones(r, device=DEV, dtype=torch.int32)
    cap = r
    if case["tokens"]:
        # a sixteenth of the requests bring a prompt chunk, a sixteenth are finished
        kind = torch.randint(0, 16, (r,), generator=g, device=DEV)
        weight = torch.rand(r, generator=g, device=DEV) * (kind == 0)
        chunk = (weight / weight.sum().clamp_min(1e-9) * case["tokens"]).floor().to(torch.int32).clamp(max=4096)
        new = torch.where(kind == 0, chunk, torch.where(kind == 1, -1, 1)).to(torch.int32)
        cached = torch.where(kind == 0, torch.zeros_like(cached), cached)
        cap = max(case["tokens"], 1) + r
    width = -(-(max(max_len, 4096) + 1) // page)
    held = (cached + page - 1) // page
    total = r * width
    pages = torch.randperm(total, generator=g, device=DEV, dtype=torch.int32)
    col = torch.arange(width, device=DEV, dtype=torch.int32)
    first = torch.cumsum(held, 0) - held
    table = torch.where(col[None] < held[:, None], pages[(first[:, None] + col[None]).clamp(max=total - 1).long()], -1)
    ring = torch.full((total,), -1, device=DEV, dtype=torch.int32)
    taken = held.sum()
    # free pages start a third of the way into the ring and wrap around
    head = torch.full((), total // 3, device=DEV, dtype=torch.int64)
    at = torch.arange(total, device=DEV)
    n_free = total - taken
    ring[((head + at) % total)] = torch.where(at < n_free, pages[(taken + at) % total], -1)
    return {"cached": cached, "new": new, "table": table.to(torch.int32).contiguous(), "ring": ring,
            "ring_in": torch.stack([head, head + n_free]), "page": page, "cap": cap}


def _prepare_write(case, g):
    n, page = case["rows"], case["page"]
    pages = -(-n // page) + 7
    order = torch.randperm(pages, generator=g, device=DEV)
    i = torch.arange(n, device=DEV)
    slots = order[i // page] * page + i % page
    if case["pad"]:
        slots = torch.where(i % case["pad"] == case["pad"] - 1, -1, slots)
    cache = torch.randint(0, 256, (pages, page // BLOCK_TOKENS * BLOCK_BYTES), generator=g, device=DEV, dtype=torch.uint8)
    return {"rows": _latent_rows(n, g), "slots": slots, "cache": cache,
            "out": torch.empty(n, ROW, device=DEV, dtype=torch.bfloat16)}


def _prepare_attn(case, g):
    page, q, seqs = case["page"], case["queries"], case["seqs"]
    lens = torch.tensor(_lens(case), device=DEV, dtype=torch.int64)[torch.randperm(seqs, generator=g, device=DEV)]
    width = max(1, -(-max(_lens(case)) // page)) + 1
    held = (lens + page - 1) // page
    pages = int(sum(-(-v // page) for v in _lens(case))) + 3
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    col = torch.arange(width, device=DEV)
    first = torch.cumsum(held, 0) - held
    table = torch.where(col[None] < held[:, None], order[(first[:, None] + col[None]).clamp(max=pages - 1)], -1)
    cache = torch.empty(pages, page // BLOCK_TOKENS * BLOCK_BYTES, device=DEV, dtype=torch.uint8)
    blocks = cache.view(-1, BLOCK_BYTES)
    step = 8192                                     # blocks at a time: bounds the temporaries
    for b0 in range(0, blocks.shape[0], step):
        nb = min(step, blocks.shape[0] - b0)
        blocks[b0:b0 + nb] = _pack(*_quantise(_latent_rows(nb * BLOCK_TOKENS, g))).view(nb, BLOCK_BYTES)
    rows = seqs * q
    # the queries are the last q positions of their sequence; an empty one attends nothing
    positions = (lens[:, None] - q + torch.arange(q, device=DEV)[None]).clamp(min=-1).reshape(-1).contiguous()
    positions = torch.where(lens.repeat_interleave(q) == 0, -1, positions)
    return {"q_abs": torch.randn(rows, HEADS, LATENT, generator=g, device=DEV).to(torch.bfloat16),
            "q_pe": torch.randn(rows, HEADS, ROPE, generator=g, device=DEV).to(torch.bfloat16),
            "cache": cache, "table": table.to(torch.int32).contiguous(), "positions": positions, "page": page,
            "seq_rows": torch.arange(seqs, device=DEV, dtype=torch.int32).repeat_interleave(q).contiguous(),
            "max_len": max(_lens(case)), "out": torch.empty(rows, HEADS, LATENT, device=DEV, dtype=torch.bfloat16)}


def _prepare_lora(case, g):
    t, na, r, k, n = case["rows"], case["adapters"], case["rank"], case["k"], case["n"]
    i = torch.arange(t, device=DEV)
    ids = torch.where(i % 8 == 7, -1, i % na).to(torch.int32)[torch.randperm(t, generator=g, device=DEV)]

    def bf(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)
    return {"x": bf(t, k), "w": bf(n, k, std=0.02), "a": bf(na, r, k, std=k ** -0.5), "b": bf(na, n, r, std=0.02),
            "ids": ids.contiguous(), "ranks": torch.tensor(_ranks(case), device=DEV, dtype=torch.int32),
            "scales": torch.rand(na, generator=g, device=DEV) + 1.0,
            "out": torch.empty(t, n, device=DEV, dtype=torch.bfloat16)}


def prepare(case, seed):
    make = {"plan": _prepare_plan, "write": _prepare_write, "attn": _prepare_attn, "lora": _prepare_lora}[case["op"]]
    return {"op": case["op"], **make(case, _gen(seed))}


# ------------------------------------------------------------------ the cache format, plain
def _p():
    return torch.arange(BLOCK_TOKENS, device=DEV)


def _group_place():
    """[16 tokens, 16 groups]: where a token's row holds group c."""
    p, c = _p(), torch.arange(16, device=DEV)
    return c[None] ^ (2 * (p & 1) + 4 * (((p >> 1) ^ (p >> 2)) & 1))[:, None]


def _scale_place():
    p = _p()
    return 4 * (p & 3) + (p >> 2)


def _rope_place():
    return torch.arange(8, device=DEV)[None] ^ (_p() & 4)[:, None]


def _nibble_dims():
    """Nibble n of a word holds dim order[n] of its 8."""
    return torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=DEV)


def _scale_of(code):
    return (code.to(torch.int32) << 7).to(torch.int16).view(torch.float16).float()


def _quantise(rows):
    """bf16 rows [N, 576] -> nibbles [N, 16, 32] (0..15), scale codes [N, 16], roped dims [N, 64].
    scale = max |x| / 7 to 3 mantissa bits (nearest, ties to even), value = round(x / scale)."""
    x = rows[:, :LATENT].float().view(-1, 16, 32)
    # by a tensor on the device: a division by a plain number is done as a product with its
    # rounded reciprocal, and max |x| / 7 is often halfway between two scales
    s = x.abs().amax(-1) / torch.full((), 7.0, device=DEV)
    bits = s.view(torch.int32)
    normal = ((bits + 0x7FFFF + ((bits >> 20) & 1)) >> 20) - (112 << 3)
    code = torch.where(s < 2.0 ** -14, torch.round(s * 2.0 ** 17).to(torch.int32), normal).clamp(max=MAX_CODE)
    s = _scale_of(code)[..., None]
    q = torch.where(s > 0, torch.round(x / s).clamp(-8, 7), 0.0)
    return (q + 8).to(torch.uint8), code.to(torch.uint8), rows[:, LATENT:]


def _token_bytes(nibbles, code, rope):
    """A token's 256 + 16 + 128 bytes in the order of its groups and dims."""
    n = nibbles.shape[0]
    word = nibbles.view(n, 16, 4, 8)[..., _nibble_dims()].view(n, 16, 4, 4, 2)
    lat = (word[..., 0] | (word[..., 1] << 4)).view(n, 256)
    return torch.cat([lat, code, rope.contiguous().view(torch.uint8)], 1)


def _token_places():
    """[16 tokens, 400]: the block byte that holds each byte of a token."""
    p, b = _p()[:, None], torch.arange(16, device=DEV)
    lat = (p[..., None] * 256 + _group_place()[..., None] * 16 + b).view(BLOCK_TOKENS, 256)
    sc = 4096 + 16 * b[None] + _scale_place()[:, None]
    rope = (4352 + p[..., None] * 128 + _rope_place()[..., None] * 16 + b).view(BLOCK_TOKENS, 128)
    return torch.cat([lat, sc, rope], 1)


def _pack(nibbles, code, rope):
    """Consecutive tokens (a multiple of 16) -> blocks [N / 16, 6400]."""
    n = nibbles.shape[0] // BLOCK_TOKENS
    out = torch.empty(n, BLOCK_BYTES, device=DEV, dtype=torch.uint8)
    out[:, _token_places().view(-1)] = _token_bytes(nibbles, code, rope).view(n, BLOCK_BYTES)
    return out


def _values(token_bytes):
    """Token bytes [..., 400] -> fp32 latent [..., 512] and roped dims [..., 64]."""
    lat, code, rope = token_bytes[..., :256], token_bytes[..., 256:272], token_bytes[..., 272:]
    nib = torch.stack([lat & 15, lat >> 4], -1).view(*lat.shape[:-1], 16, 4, 8)
    nib = nib[..., torch.argsort(_nibble_dims())].reshape(*lat.shape[:-1], 16, 32)
    val = (nib.float() - 8) * _scale_of(code)[..., None]
    return val.view(*lat.shape[:-1], LATENT), rope.contiguous().view(torch.bfloat16).float()


# ------------------------------------------------------------------ plain forms
def _plain_plan(s):
    cached, new, page, table, ring = s["cached"].long(), s["new"].long(), s["page"], s["table"], s["ring"]
    r, width = table.shape
    size = ring.numel()
    head, tail = s["ring_in"][0], s["ring_in"][1]
    fresh = new.clamp(min=0)
    held = (cached + page - 1) // page
    need = torch.where(new >= 0, (cached + fresh + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0)
    served = (new >= 0) & ((need == 0) | (upto <= tail - head))
    taken = torch.where(served & (need > 0), upto, 0).amax()
    col = torch.arange(width, device=DEV)[None]
    mine = served[:, None] & (col >= held[:, None]) & (col < (held + need)[:, None])
    at = (head + (upto - need)[:, None] + col - held[:, None]) % size
    table.copy_(torch.where(mine, ring[at], table))
    back = torch.where(new < 0, held, 0)
    back_upto = torch.cumsum(back, 0)
    gone = col < back[:, None]
    to = torch.where(gone, (tail + (back_upto - back)[:, None] + col) % size, size)
    ring.copy_(torch.cat([ring, ring[:1]]).scatter(0, to.view(-1), table.view(-1))[:size])
    cu = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), torch.cumsum(fresh, 0)])
    t = torch.arange(s["cap"], device=DEV)
    row = torch.searchsorted(cu[1:], t, right=True)
    live = row < r
    row = row.clamp(max=r - 1)
    pos = cached[row] + t - cu[row]
    slot = table[row, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    lens = torch.where(new < 0, 0, torch.where(served, cached + fresh, cached))
    counts = torch.stack([cu[-1], taken, back_upto[-1], ((new >= 0) & ~served).sum()])
    return {"table": table, "ring": ring, "ring_out": torch.stack([head + taken, tail + back_upto[-1]]),
            "token_row": torch.where(live, row, -1).to(torch.int32), "positions": torch.where(live & served[row], pos, -1),
            "slots": torch.where(live & served[row], slot, -1), "cu_new": cu.to(torch.int32),
            "lens": lens.to(torch.int32), "counts": counts.to(torch.int32)}


def _plain_write(s):
    cache, slots = s["cache"].view(-1), s["slots"]
    live = slots >= 0
    at = slots.clamp(min=0)
    place = (at // BLOCK_TOKENS * BLOCK_BYTES)[:, None] + _token_places()[at % BLOCK_TOKENS]
    cache[place[live].view(-1)] = _token_bytes(*_quantise(s["rows"]))[live].view(-1)
    lat, rope = _values(cache[place])
    return torch.where(live[:, None], torch.cat([lat, rope], 1), 0.0).to(torch.bfloat16)


def _plain_attn(s):
    page, n_blk = s["page"], -(-max(1, s["max_len"]) // BLOCK_TOKENS)
    seq = s["seq_rows"].long()
    blk = torch.arange(n_blk, device=DEV)
    per = page // BLOCK_TOKENS
    block = s["table"].long()[:, blk // per].clamp(min=0) * per + blk % per      # [sequences, blocks]
    tokens = s["cache"].view(-1, BLOCK_BYTES)[block][..., _token_places()]
    lat, rope = _values(tokens.view(block.shape[0], n_blk * BLOCK_TOKENS, 400))
    queries = seq.numel() // block.shape[0]
    q_abs, q_pe = (s[k].float().view(block.shape[0], queries * HEADS, -1) for k in ("q_abs", "q_pe"))
    score = (q_abs @ lat.transpose(1, 2) + q_pe @ rope.transpose(1, 2)) * SOFTMAX_SCALE
    pos = s["positions"].view(-1, queries).repeat_interleave(HEADS, 1)[..., None]
    seen = torch.arange(n_blk * BLOCK_TOKENS, device=DEV) <= pos
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - top), 0.0)
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    return (p @ lat).view(seq.numel(), HEADS, LATENT).to(torch.bfloat16)


def _plain_lora(s):
    x, ids = s["x"].float(), s["ids"].long()
    na, r, k = s["a"].shape
    used = torch.arange(r, device=DEV)[None] < s["ranks"][:, None]
    a = torch.where(used[..., None], s["a"].float(), 0.0)
    b = torch.where(used[:, None], s["b"].float(), 0.0) * s["scales"][:, None, None]
    mine = (ids[:, None] == torch.arange(na, device=DEV))[..., None]
    low = torch.where(mine, (x @ a.view(na * r, k).t()).view(-1, na, r), 0.0).view(-1, na * r)
    return (x @ s["w"].float().t() + low @ b.transpose(1, 2).reshape(na * r, -1)).to(torch.bfloat16)


# ------------------------------------------------------------------ one pass
def _own(s):
    ops = _ops()
    op = s["op"]
    if op == "plan":
        if "buf" not in s:
            s["buf"] = ops.page_plan_buffers(s["table"].shape[0], s["cap"], DEV)
        b = s["buf"]
        ops.page_plan(cached=s["cached"], new=s["new"], block_table=s["table"], free_ring=s["ring"], ring_in=s["ring_in"],
                      page_size=s["page"], **b)
        return {"table": s["table"], "ring": s["ring"],
                **{k: b[k] for k in ("ring_out", "token_row", "positions", "slots", "cu_new", "lens", "counts")}}
    if op == "write":
        ops.latent4_write(rows=s["rows"], slots=s["slots"], cache=s["cache"])
        return ops.latent4_read(cache=s["cache"], slots=s["slots"], out=s["out"])
    if op == "attn":
        if "ws" not in s:
            s["ws"] = ops.mla_q4_workspace(s["q_abs"].shape[0], DEV)
        return ops.mla_decode_q4(q_abs=s["q_abs"], q_pe=s["q_pe"], cache=s["cache"], block_table=s["table"],
                                 positions=s["positions"], seq_rows=s["seq_rows"], page_size=s["page"],
                                 softmax_scale=SOFTMAX_SCALE, o_lat=s["out"], **s["ws"])
    if "ws" not in s:
        s["ws"] = ops.lora_workspace(s["x"].shape[0], s["w"].shape[0], s["w"].shape[1], s["a"].shape[1], DEV)
    return ops.lora_linear(x=s["x"], w=s["w"], a=s["a"], b=s["b"], ids=s["ids"], ranks=s["ranks"], scales=s["scales"],
                           y=s["out"], **s["ws"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "write": _plain_write, "attn": _plain_attn, "lora": _plain_lora}[state["op"]](state)


# ------------------------------------------------------------------ 64-bit values
def _exact_token(block_bytes, p):
    """Token p's latent and roped dims from its block's bytes, straight from the format."""
    d = torch.arange(LATENT, device=DEV)
    group, word, j = d // 32, d % 32 // 8, d % 8
    nib = j // 2 + 4 * (j % 2)
    f = 2 * (p % 2) + 4 * ((p // 2 % 2) ^ (p // 4 % 2))
    byte = block_bytes[..., 256 * p + 16 * (group ^ f) + 4 * word + nib // 2].to(torch.int64)
    q = byte // 16 ** (nib % 2) % 16 - 8
    code = block_bytes[..., 4096 + 16 * group + 4 * (p % 4) + p // 4].to(torch.int64)
    e, m = code // 8, (code % 8).double()
    scale = torch.where(e == 0, m * 2.0 ** -17, (1 + m / 8) * torch.exp2((e - 15).double()))
    r = torch.arange(ROPE, device=DEV)
    at = 4352 + 128 * p + 16 * (r // 8 ^ (4 * (p // 4 % 2))) + 2 * (r % 8)
    hi, lo = block_bytes[..., at + 1].to(torch.int32), block_bytes[..., at].to(torch.int32)
    rope = ((hi << 24) | (lo << 16)).view(torch.float32).double()
    return q.double() * scale, rope


def _exact_write(s):
    x = s["rows"][:, :LATENT].double().view(-1, 16, 32)
    s0 = x.abs().amax(-1, keepdim=True) / 7
    e = torch.floor(torch.log2(s0.clamp(min=2.0 ** -14)))
    step = torch.exp2(e - 3)
    scale = (torch.round(s0 / step) * step).clamp(max=60.0)
    q = torch.where(scale > 0, torch.round(x / scale).clamp(-8, 7), 0.0)
    out = torch.cat([(q * scale).view(-1, LATENT), s["rows"][:, LATENT:].double()], 1)
    return torch.where(s["slots"][:, None] >= 0, out, 0.0)


def _exact_attn(s):
    page, out = s["page"], torch.zeros(s["q_abs"].shape, device=DEV, dtype=torch.float64)
    per = page // BLOCK_TOKENS
    positions, seqs, table = s["positions"].tolist(), s["seq_rows"].tolist(), s["table"].long()
    held = {}
    for i, (pos, seq) in enumerate(zip(positions, seqs)):
        if pos < 0:
            continue
        if seq not in held:
            n = max(p for p, q in zip(positions, seqs) if q == seq) + 1
            blk = torch.arange(-(-n // BLOCK_TOKENS), device=DEV)
            data = s["cache"].view(-1, BLOCK_BYTES)[table[seq, blk // per] * per + blk % per]
            both = [_exact_token(data, p) for p in range(BLOCK_TOKENS)]
            held = {seq: [torch.stack([b[k] for b in both], 1).flatten(0, 1) for k in (0, 1)]}
        lat, rope = (v[:pos + 1] for v in held[seq])
        score = (s["q_abs"][i].double() @ lat.t() + s["q_pe"][i].double() @ rope.t()) * SOFTMAX_SCALE
        out[i] = torch.softmax(score, -1) @ lat
    return out


def _exact_lora(s):
    x = s["x"].double()
    y = x @ s["w"].double().t()
    ids, ranks = s["ids"].long(), s["ranks"].tolist()
    for a, r in enumerate(ranks):
        rows = torch.nonzero(ids == a).view(-1)
        low = x[rows] @ s["a"][a, :r].double().t()
        y[rows] += low @ s["b"][a, :, :r].double().t() * s["scales"][a].double()
    return y


def exact(case, seed):
    if case["op"] == "plan":
        return None                  # whole numbers: equal or wrong
    return {"write": _exact_write, "attn": _exact_attn, "lora": _exact_lora}[case["op"]](prepare(case, seed))
