"""64-bit restatements of the paged 4-bit serving operators, written from their definitions in
include/dsv2.h (CPU, sequential where order matters).  Test-only."""
from __future__ import annotations

import torch

BLOCK_TOKENS, BLOCK_BYTES, MAX_CODE = 16, 6400, 167


def scale_value(code: torch.Tensor) -> torch.Tensor:
    """The scale of a code: 5 exponent bits, 3 mantissa bits, bias 15, subnormals at exponent 0."""
    e, m = (code.long() >> 3), (code.long() & 7).double()
    return torch.where(e == 0, m * 2.0 ** -17, (1 + m / 8) * torch.exp2((e - 15).double()))


SCALES = scale_value(torch.arange(MAX_CODE + 1))


def scale_code(amax: torch.Tensor) -> torch.Tensor:
    """Nearest scale to amax / 7 by search over every code; an even code on a tie."""
    s = amax.double() / 7
    s = s.clamp(max=float(SCALES[-1]))                     # infinities saturate
    d = (s[..., None] - SCALES).abs()
    best = d.min(-1, keepdim=True).values
    codes = torch.arange(MAX_CODE + 1)
    tied = torch.where(d == best, codes, torch.full_like(codes, 1 << 20))
    lo = tied.min(-1).values
    hi = torch.where(d == best, codes, torch.full_like(codes, -1)).max(-1).values
    return torch.where((lo != hi) & (lo % 2 == 1), hi, lo)


def quantise(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 rows [n, 576] -> integers [n, 512] in -8..7 and scale codes [n, 16]."""
    x = rows[:, :512].double().view(-1, 16, 32)
    finite_max = torch.where(x.isnan(), 0.0, x.abs()).amax(-1)
    code = scale_code(finite_max)
    s = scale_value(code)[..., None]
    v = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)).clamp(-8, 7), 0.0)
    v = torch.where(x.isnan(), 0.0, v)
    return v.view(-1, 512), code


def values(rows: torch.Tensor) -> torch.Tensor:
    """What the cache holds for bf16 rows [n, 576], in 64 bits."""
    v, code = quantise(rows)
    lat = (v.view(-1, 16, 32) * scale_value(code)[..., None]).view(-1, 512)
    return torch.cat([lat, rows[:, 512:].double()], 1)


def token_bytes(rows: torch.Tensor, tok: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(bytes [n, 400], their offsets in the 6400-byte block [n, 400]) of rows at tokens tok of
    their blocks, from the byte layout in include/dsv2.h."""
    v, code = quantise(rows)
    n = rows.shape[0]
    nib = (v + 8).to(torch.uint8).view(n, 16, 4, 8)          # group, word, dim of the word
    data = torch.zeros(n, 400, dtype=torch.uint8)
    off = torch.zeros(n, 400, dtype=torch.int64)
    p = tok.long()
    f = 2 * (p & 1) + 4 * (((p >> 1) ^ (p >> 2)) & 1)
    k = 0
    for c in range(16):
        for w in range(4):
            for byte in range(4):                            # nibbles 2 byte and 2 byte + 1
                n0, n1 = 2 * byte, 2 * byte + 1
                d0, d1 = (2 * i if i < 4 else 2 * (i - 4) + 1 for i in (n0, n1))
                data[:, k] = nib[:, c, w, d0] | (nib[:, c, w, d1] << 4)
                off[:, k] = 256 * p + 16 * (c ^ f) + 4 * w + byte
                k += 1
    for c in range(16):
        data[:, k] = code[:, c].to(torch.uint8)
        off[:, k] = 4096 + 16 * c + 4 * (p & 3) + (p >> 2)
        k += 1
    rope = rows[:, 512:].contiguous().view(torch.uint8).view(n, 128)
    for i in range(128):
        j = i // 16
        data[:, k] = rope[:, i]
        off[:, k] = 4352 + 128 * p + 16 * (j ^ (p & 4)) + i % 16
        k += 1
    return data, off


def write(rows: torch.Tensor, slots: torch.Tensor, cache: torch.Tensor) -> None:
    """Rows into their slots of a CPU cache (uint8), in place."""
    live = slots >= 0
    rows, slots = rows[live], slots[live].long()
    data, off = token_bytes(rows, slots % BLOCK_TOKENS)
    cache.view(-1)[(slots // BLOCK_TOKENS)[:, None] * BLOCK_BYTES + off] = data


def page_plan(cached, new, table, ring, ring_in, page, capacity):
    """Sequential form of dsv2_page_plan; table [R, width] and ring are lists changed in place.
    Returns a dict of lists."""
    head, tail = ring_in
    avail, size = tail - head, len(ring)
    asked = taken = put = tokens = deferred = 0
    out = {"token_row": [], "positions": [], "slots": [], "cu_new": [0], "lens": []}
    returned = []
    for r, (c, n) in enumerate(zip(cached, new)):
        if n < 0:
            returned += table[r][:-(-c // page)]
            out["lens"].append(0)
            out["cu_new"].append(tokens)
            continue
        held, want = -(-c // page), -(-(c + n) // page)
        wide = want > len(table[r])
        need = 0 if wide else want - held
        asked += need
        served = not wide and tokens + n <= capacity and (need == 0 or asked <= avail)
        if served:
            for i in range(need):
                table[r][held + i] = ring[(head + asked - need + i) % size]
            if need:
                taken = asked
        deferred += not served
        for i in range(n):
            if tokens + i < capacity:
                pos = c + i
                out["token_row"].append(r)
                out["positions"].append(pos if served else -1)
                out["slots"].append(table[r][pos // page] * page + pos % page if served else -1)
        tokens += n
        out["lens"].append(c + n if served else c)
        out["cu_new"].append(tokens)
    for pg in returned:
        ring[(tail + put) % size] = pg
        put += 1
    for k in ("token_row", "positions", "slots"):
        out[k] += [-1] * (capacity - len(out[k]))
    out["ring_out"] = [head + taken, tail + put]
    out["counts"] = [tokens, taken, put, deferred]
    return out


def attention(q_abs, q_pe, latent, rope, scale):
    """One row: q_abs [16, 512], q_pe [16, 64], latent [n, 512], rope [n, 64] (64-bit).  Returns
    the output and sum_s p[s] |latent[s]|, by which rounding errors are bounded."""
    if latent.shape[0] == 0:
        z = torch.zeros(16, 512, dtype=torch.float64)
        return z, z, 0.0
    s = (q_abs @ latent.t() + q_pe @ rope.t()) * scale
    p = torch.softmax(s, -1)
    terms = (q_abs.abs() @ latent.abs().t() + q_pe.abs() @ rope.abs().t()) * abs(scale)
    return p @ latent, p @ latent.abs(), float(terms.max())


def lora(x, w, a, b, ids, ranks, scales):
    """(y, sum_j |low_j B_j|, sum_k |x w|) in 64 bits; w may be None."""
    x = x.double()
    n = b.shape[1]
    y = torch.zeros(x.shape[0], n, dtype=torch.float64) if w is None else x @ w.double().t()
    mag = torch.zeros_like(y) if w is None else x.abs() @ w.double().abs().t()
    low_mag = torch.zeros(x.shape[0], n, dtype=torch.float64)
    for t, i in enumerate(ids):
        if i < 0:
            continue
        r = int(ranks[i])
        low = (x[t] @ a[i, :r].double().t()) * float(scales[i])
        y[t] += low @ b[i, :, :r].double().t()
        low_mag[t] = low.abs() @ b[i, :, :r].double().abs().t()
        # fp32 sums of low: k products each
        mag[t] += (x[t].abs() @ a[i, :r].double().abs().t() * abs(float(scales[i]))) @ b[i, :, :r].double().abs().t()
    return y, low_mag, mag
