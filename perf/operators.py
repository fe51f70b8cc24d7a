"""Cases of the operators that a serving program calls on its own device buffers: appending to and attending over a paged cache held in
8 bits, products with 4-bit weights, log probabilities of given tokens. Each case is one call of one operator as such a program makes it, or
(`run` with `own` false) the same computed by elementary operations in 32 bits.

Sizes are those of GPT-2 (12 heads of 64, width 768, 50257 tokens; XL: width 1600), of this repository's layered models (32000 tokens), or
generic. Lengths, page tables and row counts come from the case alone, values from the seed.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def _append(name, dtype, seqs, rows, context, heads, kv_heads, dim, rot, page, ragged):
    """`rows`: the most new tokens of a sequence; `context`: the most tokens it has after the call; `ragged`: the others have fewer of both."""
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "rows": rows, "context": context, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "page": page, "ragged": ragged}


def _attend(name, dtype, seqs, rows, context, heads, kv_heads, dim, page, ragged, window=0, keep=0):
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "rows": rows, "context": context, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "ragged": ragged, "window": window, "keep": keep}


def _q4(name, dtype, m, n, k, group, bias):
    return {"name": name, "op": "q4", "dtype": dtype, "m": m, "n": n, "k": k, "group": group, "bias": bias}


def _logprobs(name, dtype, rows, vocab, top):
    return {"name": name, "op": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top}


def listed():
    return [
        # one user's next token, GPT-2 small's heads, no rotation: nothing but latency
        _append("append_one", "f32", 1, 1, 300, 12, 12, 64, 0, 32, False),
        # a loaded server's step: one token for each of 64 sequences of different lengths, grouped heads, queries rotated on the way
        _append("append_step_64", "bf16", 64, 1, 4000, 32, 8, 128, 128, 64, True),
        # prompts of different lengths at once, half of each head rotated, head size that is no power of two
        _append("append_prompts_8", "bf16", 8, 2047, 2047, 20, 4, 96, 48, 64, True),
        # one user's next token, GPT-2 small's heads
        _attend("attend_one", "f32", 1, 1, 777, 12, 12, 64, 32, False),
        # a loaded server's step
        _attend("attend_step_64", "bf16", 64, 1, 2900, 32, 8, 128, 64, True),
        # two long documents, token by token
        _attend("attend_long", "bf16", 2, 1, 131000, 32, 4, 128, 64, False),
        # portions of two prompts behind what the cache holds of them
        _attend("attend_portions", "bf16", 2, 1500, 4100, 32, 8, 128, 64, True),
        # GPT-2 small's attention input product for one token
        _q4("q4_one", "f32", 1, 2304, 768, 64, True),
        # GPT-2 XL's first feed-forward product for eight sequences
        _q4("q4_step_8", "bf16", 8, 6400, 1600, 64, True),
        # the widest product of a large layer for a step of 16 sequences
        _q4("q4_wide_16", "bf16", 16, 28672, 8192, 128, False),
        # the end of a step of 8 sequences: the drawn tokens' log probabilities and five alternatives each
        _logprobs("logprobs_step_8", "f32", 8, 50257, 5),
        # scoring of given text
        _logprobs("logprobs_score", "bf16", 4096, 32000, 0),
    ]


def _log_int(rng, low, high):
    high = max(low, high)
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "q4", "logprobs"))
    dtype = rng.choice(("f32", "bf16"))
    if op in ("append", "attend"):
        dim = rng.choice((32, 64, 64, 80, 96, 128, 128, 160, 256))
        kv_heads, group = rng.choice((1, 2, 4, 8, 12)), rng.choice((1, 2, 4, 5, 8, 16))
        page, ragged = rng.choice((16, 32, 64)), rng.random() < 0.7
        seqs = rng.choice((1, _log_int(rng, 2, 8), _log_int(rng, 9, 96)))
        each = kv_heads * dim * seqs
    if op == "append":
        rows = rng.choice((1, 1, _log_int(rng, 2, 2000)))
        rows = max(1, min(rows, 2047 * 8 * 24 * 96 // (each * (group + 1) * 3)))
        context = rows + rng.choice((0, _log_int(rng, 1, max(1, 20000000 // each))))
        case = _append("", dtype, seqs, rows, context, kv_heads * group, kv_heads, dim, rng.choice((0, dim, dim // 2)), page, ragged)
    elif op == "attend":
        if rng.random() < 0.6:
            rows, context = rng.choice((1, 1, 1, 4)), _log_int(rng, 1, min(131000, 120000000 // each))
        else:
            rows = _log_int(rng, 5, 2000)
            context = rows + rng.choice((0, _log_int(rng, 1, 4000)))
            while rows * context * each * group > 1500 * 3400 * 4096 * (0.5 if dtype == "f32" else 1):
                rows, context = rows // 2 + 1, context // 2 + 1
            while rows * each * group > 6000000:
                rows, context = rows // 2 + 1, context - rows + rows // 2 + 1
        window = rng.choice((0, 0, _log_int(rng, 1, max(1, context))))
        keep = rng.choice((0, 4, 70)) if window else 0
        case = _attend("", dtype, seqs, min(rows, context), context, kv_heads * group, kv_heads, dim, page, ragged, window, keep)
    elif op == "q4":
        m, k = _log_int(rng, 1, 16), _log_int(rng, 64, 16384)
        case = _q4("", dtype, m, _log_int(rng, 16, min(32000, 16384 * 8192 // k)), k, rng.choice((64, 128)), rng.random() < 0.5)
    else:
        vocab = _log_int(rng, 1000, 160000)
        rows = _log_int(rng, 1, 4000 * 32000 // (vocab * (2 if dtype == "f32" else 1)))
        case = _logprobs("", dtype, rows, vocab, rng.choice((0, 1, 5, 20)))
    del case["name"]
    return case


def _shape_of(case):
    """New rows and tokens (after the call) of every sequence, from the case alone."""
    n, c, r = case["seqs"], case["context"], case["rows"]
    if not case["ragged"]:
        return [r] * n, [c] * n
    rows = [max(1, r - (i * 37 + 11 * i * i) % max(1, r // 2 + 1)) for i in range(n)]
    return rows, [max(rows[i], c - (i * 731 + 97 * i * i) % max(1, c - c // 8)) for i in range(n)]


def _padded(dim):
    return -(-dim // 64) * 64


def _cdiv(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _prepare_cache(case, g, rows, lens):
    """A pool as earlier appends left it: codes of normal values, power-of-two scales, pages in random order."""
    page, kvh, dim, dp = case["page"], case["kv_heads"], case["dim"], _padded(case["dim"])
    per_seq = _cdiv(max(lens), page)
    used = [_cdiv(n, page) for n in lens]
    pages = sum(used) + 2
    pool = torch.empty(pages, kvh, 2 * page * dp, dtype=torch.uint8, device="cuda")
    for i in range(0, pages, 512):  # in pieces: the values of a whole pool would be four times its bytes
        part = torch.randn(min(512, pages - i), kvh, 2 * page * dp, generator=g, device="cuda").mul_(100).clamp_(-448, 448)
        if dp > dim:
            part[..., :page * dp].view(-1, kvh, page, dp)[..., dim:] = 0
            part[..., page * dp:].view(-1, kvh, dp, page)[..., dim:, :] = 0
        pool[i:i + 512] = part.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.exp2(torch.randint(-8, -5, (pages, kvh, 2), generator=g, device="cuda").float())
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((len(lens), per_seq), -1, dtype=torch.int32), 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    one = all(n == 1 for n in rows)
    return {"pool": pool, "scales": scales, "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "longest": max(lens),
            "spare": order[-1:].long().cuda(), "row_start": None if one else torch.tensor(starts, dtype=torch.int32, device="cuda"), "rows": starts[-1], "max_rows": max(rows)}


def prepare(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] in ("append", "attend"):
        rows, lens = _shape_of(case)
        s.update(_prepare_cache(case, g, rows, lens))
        h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
        if case["op"] == "append":
            # the product in front leaves queries, keys and values of a token side by side
            s["qkv"] = (normal(s["rows"], h + 2 * kvh, d) * 1.5).to(dtype)
            s["q_out"] = torch.empty(s["rows"], h, d, dtype=dtype, device="cuda") if case["rot"] else None
        else:
            s["q"] = normal(s["rows"], h, d).to(dtype)
            s["out"] = torch.empty_like(s["q"])
    elif case["op"] == "q4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        nt, kt = _cdiv(n, 16), _cdiv(k, 64)
        # weights as the quantiser lays them out: tiles of 16 outputs x 64 inputs, 8 in the places behind the matrix (the code of zero)
        codes = torch.randint(1, 16, (nt * 16, kt * 64), generator=g, device="cuda", dtype=torch.uint8)
        codes[n:] = 8
        codes[:, k:] = 8
        c = codes.view(nt, 2, 8, kt, 4, 2, 8)[..., [0, 2, 4, 6, 1, 3, 5, 7]].view(nt, 2, 8, kt, 4, 2, 4, 2).permute(0, 3, 2, 4, 1, 5, 6, 7)
        s["packed"] = (c[..., 0] | c[..., 1] << 4).contiguous().view(nt, kt, 512)
        s["scales"] = (torch.rand(_cdiv(k, group), nt * 16, generator=g, device="cuda") * 0.01 + 0.002).to(torch.bfloat16)
        s["scales"][:, n:] = 0
        s["x"] = normal(m, k).to(dtype)
        s["bias"] = normal(n).to(dtype) if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=dtype, device="cuda")
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = (normal(rows, vocab) * 2.5).to(dtype)
        s["logits"][:, -max(1, vocab // 100):] = -math.inf  # entries that a filter took out
        s["targets"] = torch.randint(0, vocab - max(1, vocab // 100), (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["logprobs"], s["entropy"] = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
        s["top_ids"] = torch.empty(rows, top, dtype=torch.int32, device="cuda") if top else None
        s["top_logprobs"] = torch.empty(rows, top, dtype=torch.float32, device="cuda") if top else None
    if case["op"] in ("append", "attend") and own:
        s["cache"], s["workspace"] = _own_cache(s)
    return s


def _own_cache(s):
    import puppygrad_b200 as pg

    case = s["case"]
    cache = pg.Kv8Cache(s["pool"], s["scales"], s["table"], page_tokens=case["page"], head_dim=case["dim"])
    if case["op"] == "append":
        return cache, None
    size = cache.workspace_bytes(s["rows"], case["heads"], s["q"].dtype)
    return cache, torch.zeros(size, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _own_append(s):
    c = s["case"]
    h, kvh = c["heads"], c["kv_heads"]
    q, k, v = s["qkv"][:, :h], s["qkv"][:, h:h + kvh], s["qkv"][:, h + kvh:]
    stream = torch.cuda.current_stream().cuda_stream
    if c["rot"]:
        s["cache"].append(k, v, s["lens"], row_start=s["row_start"], q=q, q_out=s["q_out"], rot_dims=c["rot"], stream=stream)
    else:
        s["cache"].append(k, v, s["lens"], row_start=s["row_start"], stream=stream)
    return _appended(s)


def _appended(s):
    out = [s["pool"].view(torch.float8_e4m3fn), s["scales"]]
    return out + [s["q_out"]] if s["q_out"] is not None else out


def _own_attend(s):
    c = s["case"]
    s["cache"].attention(s["q"], s["out"], s["lens"], s["workspace"], row_start=s["row_start"], max_rows=s["max_rows"], window=c["window"],
                         keep_first=c["keep"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_q4(s):
    import puppygrad_b200 as pg

    pg.linear_q4(s["x"], s["packed"], s["scales"], s["out"], s["case"]["group"], bias=s["bias"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_logprobs(s):
    import puppygrad_b200 as pg

    pg.token_logprobs(s["logits"], s["targets"], s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"],
                      stream=torch.cuda.current_stream().cuda_stream)
    return _scored(s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"])


def _scored(logprobs, entropy, ids, values):
    return [logprobs, entropy] if ids is None else [logprobs, entropy, ids, values]


# ------------------------------------------------------------------ the plain forms
def _places(s):
    """(sequence, index among its new rows, position) of every row."""
    n = s["lens"].numel()
    start = s["row_start"].long() if s["row_start"] is not None else torch.arange(n + 1, device="cuda")
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), row, right=True)
    j = row - start[b]
    return b, j, s["lens"].long()[b] - (start[b + 1] - start[b]) + j


def _rotate(x, pos, rot, base=10000.0):
    """The first `rot` entries of every head, entry i with entry i + rot / 2; angles in 64 bits."""
    if not rot:
        return x
    half = rot // 2
    angle = pos.double()[:, None] * base ** (-2.0 / rot * torch.arange(half, dtype=torch.float64, device="cuda"))
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat((a * c - b * sn, b * c + a * sn, x[..., rot:]), -1)


def _need(x):
    """The power of two that brings the largest magnitude of each row of x to at most 448 (not below 2^-100)."""
    mantissa, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(mantissa > 0, e - 9 + (mantissa > 0.875), -100).clamp(min=-100)
    return torch.ldexp(torch.ones_like(mantissa), e)


def _plain_append(s):
    c = s["case"]
    h, kvh, d, p, dp = c["heads"], c["kv_heads"], c["dim"], c["page"], _padded(c["dim"])
    b, j, pos = _places(s)
    x = s["qkv"].float()
    k, v = _rotate(x[:, h:h + kvh], pos, c["rot"]), x[:, h + kvh:]
    if s["q_out"] is not None:
        s["q_out"].copy_(_rotate(x[:, :h], pos, c["rot"]).to(s["q_out"].dtype))
    kv = torch.stack((k, v), 2)  # [rows, kv heads, 2, dim]
    # the pages that get tokens: a list of `most` for every sequence, filled up with a page that no sequence has
    most = (s["max_rows"] + p - 2) // p + 1
    starts = torch.full_like(s["lens"], c["context"] + 1, dtype=torch.long).scatter_reduce(0, b, pos, "amin")
    slot = starts[:, None] // p + torch.arange(most, device="cuda")
    live = slot * p < s["lens"][:, None]
    pages = torch.where(live, s["table"].long().gather(1, slot.clamp(max=s["table"].shape[1] - 1)), s["spare"]).flatten()
    at, off = b * most + pos // p - starts[b] // p, pos % p  # the row's page in that list, its place in the page
    # scales: what the new tokens need, and what the page has where it holds earlier tokens
    first = torch.where(live, (starts[:, None] - slot * p).clamp(min=0), p).flatten()
    need = torch.zeros(pages.numel(), kvh, 2, device="cuda").index_reduce(0, at, _need(kv), "amax", include_self=True)
    held = s["scales"][pages]
    old = torch.where((first > 0)[:, None, None], held, 0.0)
    new = torch.where(live.flatten()[:, None, None], torch.maximum(need, old), held)
    ratio = torch.where(live.flatten()[:, None, None], old / new, 1.0)
    # earlier tokens of the page in the new scale
    pool = s["pool"].view(torch.float8_e4m3fn)
    codes = pool[pages].float()
    kc, vc = codes[..., :p * dp].unflatten(-1, (p, dp)), codes[..., p * dp:].unflatten(-1, (dp, p))
    before = torch.arange(p, device="cuda") < first[:, None]
    kc = torch.where(before[:, None, :, None], kc * ratio[:, :, 0, None, None], kc)
    vc = torch.where(before[:, None, None, :], vc * ratio[:, :, 1, None, None], vc)
    # the new tokens
    row = torch.nn.functional.pad(kv / new[at][..., None], (0, dp - d))
    kc[at, :, off] = row[:, :, 0]
    vc[at, :, :, off] = row[:, :, 1]
    s["pool"][pages] = torch.cat((kc.flatten(2), vc.flatten(2)), -1).to(torch.float8_e4m3fn).view(torch.uint8)
    s["scales"][pages] = new
    return _appended(s)


def _plain_attend(s):
    c = s["case"]
    h, kvh, d, p, dp, n = c["heads"], c["kv_heads"], c["dim"], c["page"], _padded(c["dim"]), s["max_rows"]
    b, j, pos = _places(s)
    seqs, used = s["lens"].numel(), _cdiv(s["longest"], p)
    table = s["table"].long()[:, :used].clamp(min=0)
    codes, scales = s["pool"].view(torch.float8_e4m3fn)[table], s["scales"][table]  # [seqs, pages, kv heads, ...]
    k = codes[..., :p * dp].unflatten(-1, (p, dp))[..., :d].float() * scales[..., 0, None, None]
    v = codes[..., p * dp:].unflatten(-1, (dp, p))[..., :d, :].float() * scales[..., 1, None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(seqs, kvh, d, used * p)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kvh, used * p, d)
    q = torch.zeros(seqs, n, h, d, device="cuda")
    q[b, j] = s["q"].float()
    q = q.view(seqs, n, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, h // kvh * n, d)
    score = (q @ k * d ** -0.5).view(seqs, kvh, h // kvh, n, used * p)
    at = torch.full((seqs, n), -1, device="cuda")
    at[b, j] = pos
    key = torch.arange(used * p, device="cuda")
    seen = key <= at[..., None]
    if c["window"]:
        seen &= (key > at[..., None] - c["window"]) | (key < c["keep"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    out = e.view(seqs, kvh, h // kvh * n, used * p) @ v
    out = torch.where(total > 0, out.view(seqs, kvh, h // kvh, n, d) / total, 0.0)
    s["out"].copy_(out.permute(0, 3, 1, 2, 4).reshape(seqs, n, h, d)[b, j])
    return s["out"]


def _plain_q4(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    nt, kt = s["packed"].shape[:2]
    p = s["packed"].view(nt, kt, 8, 4, 2, 2, 4)
    w = torch.stack((p & 15, p >> 4), -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]].permute(0, 4, 2, 1, 3, 5, 6).reshape(nt * 16, kt * 64)
    w = w[:n, :k].float() - 8
    w *= s["scales"].float().t()[:n].repeat_interleave(group, 1)[:, :k]
    out = s["x"].float() @ w.t()
    if s["bias"] is not None:
        out += s["bias"].float()
    s["out"].copy_(out)
    return s["out"]


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    logprobs = d.gather(1, s["targets"].long()[:, None])[:, 0] - log_total
    entropy = log_total - torch.where(e > 0, d * e, 0.0).sum(-1) / total
    if not s["case"]["top"]:
        return _scored(logprobs, entropy, None, None)
    ids = torch.sort(x, stable=True, dim=-1, descending=True)[1][:, :s["case"]["top"]]
    return _scored(logprobs, entropy, ids.to(torch.int32), d.gather(1, ids) - log_total[:, None])


_run_own = {"append": _own_append, "attend": _own_attend, "q4": _own_q4, "logprobs": _own_logprobs}
_run_plain = {"append": _plain_append, "attend": _plain_attend, "q4": _plain_q4, "logprobs": _plain_logprobs}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        rows = sum(_shape_of(case)[0])
        kv = rows * 2 * case["kv_heads"] * case["dim"]
        q = 2 * rows * case["heads"] * case["dim"] * size if case["rot"] else 0
        return {"bytes": kv * (size + 1) + q, "flops": 0}
    if case["op"] == "attend":
        rows, lens = _shape_of(case)
        w, keep, bytes_, pairs = case["window"], case["keep"], 0, 0
        for n, length in zip(rows, lens):
            first = length - n
            low = max(0, first - w + 1) if w else 0
            bytes_ += (length - low + min(low, keep)) * 2 * case["kv_heads"] * case["dim"]
            for t in range(first, length):
                low = max(0, t - w + 1) if w else 0
                pairs += t + 1 - low + min(low, keep)
        return {"bytes": bytes_ + 2 * sum(rows) * case["heads"] * case["dim"] * size, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k / 2 + 2 * n * _cdiv(k, case["group"]) + (m * (n + k) + (n if case["bias"] else 0)) * size, "flops": 2 * m * n * k}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * vocab * size + rows * (12 + 8 * case["top"]), "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def _bytes_to_f64(b):
    """The value of every e4m3 byte, from its fields: sign, four bits of exponent (bias 7), three of mantissa."""
    b = b.long()
    e, m = b >> 3 & 15, (b & 7).double()
    value = torch.where(e > 0, (8 + m) * torch.exp2(e.double() - 10), m * 2.0 ** -9)
    return torch.where(b > 127, -value, value)


def _grid_f64(x):
    """x rounded to the nearest e4m3 value, ties to the even mantissa."""
    a = x.abs().clamp(max=448.0)
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4)
    return torch.copysign(torch.round(a / step) * step, x)


def _turn_f64(x, pos, rot):
    out, half = x.clone(), rot // 2
    for i in range(half):
        t = pos.double() * 10000.0 ** (-2.0 * i / rot)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        out[..., i] = c * x[..., i] - s * x[..., i + half]
        out[..., i + half] = s * x[..., i] + c * x[..., i + half]
    return out


def _exact_append(s):
    c = s["case"]
    h, kvh, d, p, dp = c["heads"], c["kv_heads"], c["dim"], c["page"], _padded(c["dim"])
    rows, lens = _shape_of(c)
    pool, scales, at = _bytes_to_f64(s["pool"]), s["scales"].double(), 0
    k, v = pool[..., :p * dp].unflatten(-1, (p, dp)), pool[..., p * dp:].unflatten(-1, (dp, p)).transpose(-1, -2)
    table, turned = s["table"].tolist(), []
    for i, (n, length) in enumerate(zip(rows, lens)):
        x = s["qkv"][at:at + n].double()
        pos = torch.arange(length - n, length, device="cuda")
        new_k, new_v = _turn_f64(x[:, h:h + kvh], pos, c["rot"]), x[:, h + kvh:]
        turned.append(_turn_f64(x[:, :h], pos, c["rot"]))
        at, done = at + n, 0
        while done < n:
            t = length - n + done
            g, o, m = table[i][t // p], t % p, min(n - done, p - t % p)
            for side, (held, new) in enumerate(((k, new_k), (v, new_v))):
                part = new[done:done + m].transpose(0, 1)  # [kv heads, tokens, dim]
                fraction, e = torch.frexp((part.abs().amax((1, 2)) / 448).clamp(min=2.0 ** -100))
                need = torch.ldexp(torch.ones_like(fraction), torch.where(fraction > 0.5, e, e - 1))
                scale = torch.maximum(need, scales[g, :, side]) if o else need
                if o:
                    held[g, :, :o] = _grid_f64(held[g, :, :o] * (scales[g, :, side] / scale)[:, None, None])
                held[g, :, o:o + m, :d] = _grid_f64(part / scale[:, None, None])
                held[g, :, o:o + m, d:] = 0
                scales[g, :, side] = scale
            done += m
    out = [torch.cat((k.flatten(2), v.transpose(-1, -2).flatten(2)), -1), scales]
    return out + [torch.cat(turned)] if c["rot"] else out


def _exact_attend(s):
    c = s["case"]
    h, kvh, d, p, dp = c["heads"], c["kv_heads"], c["dim"], c["page"], _padded(c["dim"])
    rows, lens = _shape_of(c)
    out, at = torch.zeros(s["rows"], h, d, dtype=torch.float64, device="cuda"), 0
    for i, (n, length) in enumerate(zip(rows, lens)):
        pages = s["table"][i, :_cdiv(length, p)].long()
        pool, scale = _bytes_to_f64(s["pool"][pages]), s["scales"][pages].double()
        k = (pool[..., :p * dp].unflatten(-1, (p, dp)) * scale[..., 0, None, None]).transpose(0, 1).flatten(1, 2)[:, :length, :d]
        v = (pool[..., p * dp:].unflatten(-1, (dp, p)) * scale[..., 1, None, None]).transpose(2, 3).transpose(0, 1).flatten(1, 2)[:, :length, :d]
        q = s["q"][at:at + n].double()
        row, key = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")
        hidden = key > row
        if c["window"]:
            hidden |= (key <= row - c["window"]) & (key >= c["keep"])
        for x in range(h):
            score = torch.softmax((q[:, x] @ k[x * kvh // h].t() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            out[at:at + n, x] = score @ v[x * kvh // h]
        at += n
    return out


def _exact_q4(s):
    c = s["case"]
    n, k, out = c["n"], c["k"], []
    tile = torch.arange(k, device="cuda")
    for r in range(0, n, 2048):
        row = torch.arange(r, min(n, r + 2048), device="cuda")[:, None]
        field = tile % 8 // 2 + tile % 2 * 4
        byte = (row % 8 * 4 + tile % 64 // 16) * 16 + row % 16 // 8 * 8 + tile % 16 // 8 * 4 + field // 2
        code = s["packed"][row // 16, tile // 64, byte].long() >> 4 * (field % 2) & 15
        out.append(s["x"].double() @ ((code - 8).double() * s["scales"][tile // c["group"], row].double()).t())
    out = torch.cat(out, 1)
    return out + s["bias"].double() if s["bias"] is not None else out


def _exact_logprobs(s):
    lp, ent, ids, values = [], [], [], []
    for x, t in zip(s["logits"].split(256), s["targets"].split(256)):
        x = x.double()
        p = x - torch.logsumexp(x, -1, keepdim=True)
        lp.append(p.gather(1, t.long()[:, None])[:, 0])
        ent.append(-(p.exp() * p.clamp(min=-1e30)).sum(-1))
        if s["case"]["top"]:
            i = torch.argsort(-x, dim=-1, stable=True)[:, :s["case"]["top"]]
            ids.append(i.to(torch.int32))
            values.append(p.gather(1, i))
    return _scored(torch.cat(lp), torch.cat(ent), torch.cat(ids) if ids else None, torch.cat(values) if values else None)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "q4": _exact_q4, "logprobs": _exact_logprobs}[case["op"]](s)
