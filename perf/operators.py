"""Cases of the quantized key/value cache: writing tokens into it, reading them back, and attention over it.

The cache holds keys and values as ggml blocks of 32 along the head (Q4_0 or Q8_0: an f16 scale and 32 codes), in pages of
`page` tokens; a token's slot is page * page size + its place in the page.  Three operators (comp_amd.kv):

    write    K, V [T][kv heads][D] (f32, f16, bf16) are quantized into the slots given for the T tokens
    read     the tokens of given slots come back as values (f32, f16, bf16)
    attend   softmax(q K^T) V for a batch of sequences whose keys lie in pages: one query token a sequence (decode),
             a few (drafted tokens), or many (a prompt, or a piece of one after a context)

A write returns what the cache then holds for its tokens, read back in f32, since that is what the codes stand for.

With `own` false, run() computes them in plain torch operations in 32 bits; with `own` true through comp_amd.kv.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32
BYTES = {"q4_0": 18, "q8_0": 34}  # a block of 32: f16 scale and codes


# ---- the cases -------------------------------------------------------------------------------------------------------


def _write(name, tokens, runs, kv_heads, dim, k_format, v_format, dtype, page=64):
    return dict(name=name, kind="write", tokens=tokens, runs=runs, kv_heads=kv_heads, dim=dim, k_format=k_format,
                v_format=v_format, dtype=dtype, page=page)  # fmt: skip


def _read(name, tokens, kv_heads, dim, k_format, v_format, dtype, page=64):
    return dict(name=name, kind="read", tokens=tokens, runs=1, kv_heads=kv_heads, dim=dim, k_format=k_format,
                v_format=v_format, dtype=dtype, page=page)  # fmt: skip


def _attend(name, batch, queries, length, heads, kv_heads, dim, k_format, v_format, dtype, ragged=False, page=64,
            softcap=0.0, window=0, prefix=0, slopes=False, lse=False):  # fmt: skip
    return dict(name=name, kind="attend", batch=batch, queries=queries, length=length, heads=heads, kv_heads=kv_heads,
                dim=dim, k_format=k_format, v_format=v_format, dtype=dtype, ragged=ragged, page=page, softcap=softcap,
                window=window, prefix=prefix, slopes=slopes, lse=lse)  # fmt: skip


def listed():
    return [
        # one decode step of 64 sequences: each writes its one new token somewhere in its own last page
        _write("write_step", 64, 64, 8, 128, "q4_0", "q4_0", "f32"),
        # a prompt of odd length that continues in the middle of a page
        _write("write_prompt", 3001, 1, 5, 128, "q8_0", "q4_0", "bf16"),
        # many prompts at once, or one very long one
        _write("write_long", 65536, 7, 8, 128, "q8_0", "q8_0", "f32"),
        # one short sequence leaves the cache (it is moved, or its attention runs elsewhere)
        _read("read_short", 1500, 8, 64, "q4_0", "q4_0", "f16"),
        # a long context leaves the cache
        _read("read_long", 49999, 8, 128, "q8_0", "q4_0", "bf16"),
        # one user's next token over a short context (f32 activations, as this package's GEMVs give them)
        _attend("step_one", 1, 1, 1000, 32, 8, 128, "q4_0", "q4_0", "f32"),
        # 16 users of unlike lengths, 1 to 5 drafted tokens each to be checked; 20 query and 5 cache heads
        _attend("step_drafts", 16, 5, 8192, 20, 5, 128, "q8_0", "q4_0", "f32", ragged=True, lse=True),
        # one user's next token over a very long context
        _attend("step_long", 1, 1, 131072, 32, 8, 128, "q4_0", "q4_0", "bf16"),
        # a full server's decode step: 64 users, lengths up to 8192
        _attend("step_batch", 64, 1, 8192, 32, 8, 128, "q4_0", "q4_0", "bf16", ragged=True),
        # as many heads in the cache as in the query, an odd number of blocks a head, scores falling with the distance
        _attend("step_heads", 8, 1, 3000, 12, 12, 96, "q8_0", "q8_0", "f16", ragged=True, page=32, slopes=True),
        # pieces of three prompts after their contexts: capped scores, a window
        _attend("chunk_window", 3, 700, 5701, 16, 8, 256, "q8_0", "q8_0", "f16", ragged=True, softcap=50.0, window=2048),
        # a whole prompt whose first 500 tokens see each other both ways
        _attend("prompt", 1, 4096, 4096, 32, 8, 128, "q4_0", "q4_0", "bf16", prefix=500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kf, vf = rng.choice([("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q8_0", "q8_0")])
    dim, dtype, page = rng.choice([64, 96, 128, 256]), rng.choice(["f32", "f16", "bf16"]), rng.choice([32, 64, 128])
    kind = rng.choice(["write", "read", "step", "step", "drafts", "chunk"])
    kv = rng.choice([1, 2, 4, 5, 8, 12])
    if kind in ("write", "read"):
        tokens = _log(rng, 1, max(1, 65536 * 8 * 128 // (kv * dim) // 2))
        case = dict(kind=kind, tokens=tokens, runs=rng.randint(1, min(tokens, 32)) if kind == "write" else 1, kv_heads=kv,
                    dim=dim, k_format=kf, v_format=vf, dtype=dtype, page=page)  # fmt: skip
        return case
    g = rng.choice([1, 2, 4, 7, 8, 16])
    if kind == "chunk":
        queries = _log(rng, 16, 2048)
        batch = rng.randint(1, 3)
        length = queries + _log(rng, 1, 4096)
        g = min(g, 4)
    else:
        queries = 1 if kind == "step" else rng.randint(2, 8)
        batch = _log(rng, 1, 64)
        length = queries + _log(rng, 1, 65536)
    # no more keys to read, and no more products, than the largest listed cases
    while batch * length * kv * dim > 20 * 8192 * 8 * 128 and length > 2 * queries:
        length = max(queries, length // 2 + 1)
    while batch * queries * length * kv * g * dim > 4096 * 2048 * 32 * 128 and kv * g > 1:
        g, kv = (max(1, g // 2), kv) if g > 1 else (g, max(1, kv // 2))
    return dict(kind="attend", batch=batch, queries=queries, length=length, heads=kv * g, kv_heads=kv, dim=dim, k_format=kf,
                v_format=vf, dtype=dtype, ragged=rng.random() < 0.6, page=page, softcap=rng.choice([0.0, 0.0, 30.0]),
                window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), prefix=rng.choice([0, 0, _log(rng, 1, length)]),
                slopes=rng.random() < 0.25, lse=rng.random() < 0.25)  # fmt: skip


# ---- what a case's sizes say before any values -----------------------------------------------------------------------


def _shape_rng(case):
    return random.Random("%d %d %d" % (case["kv_heads"], case["dim"], case.get("length", case.get("tokens"))))


def _sequences(case):
    """[(keys, queries)] of an attention case's sequences: the same for every seed."""
    r, got = _shape_rng(case), []
    for b in range(case["batch"]):
        n, q = case["length"], case["queries"]
        if case["ragged"] and b:  # the first sequence keeps the full length
            n = r.randint(max(1, n // 16), n) if b % 4 else r.randint(1, n)
            q = r.randint(1, min(q, n))
        got.append((n, q))
    return got


def _runs(case):
    """Lengths of the stretches of consecutive slots that a write or read goes to."""
    n, runs = case["tokens"], case["runs"]
    cuts = sorted(_shape_rng(case).sample(range(1, n), runs - 1)) if runs > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [n])]


def _block_bytes(case):
    """Cache bytes of one token and head, keys and values."""
    return case["dim"] // BLOCK * (BYTES[case["k_format"]] + BYTES[case["v_format"]])


def _pairs(case):
    """(visible query-key pairs, keys that some query sees) over an attention case's sequences, a head."""
    pairs = keys = 0
    for n, q in _sequences(case):
        at = torch.arange(n - q, n, dtype=torch.int64)
        hi = torch.clamp(torch.maximum(at + 1, torch.tensor(case["prefix"])), max=n)
        lo = torch.clamp(at - case["window"] + 1, min=0) if case["window"] else torch.zeros_like(at)
        pairs += int(torch.clamp(hi - lo, min=0).sum())
        keys += int(hi.max() - lo.min())
    return pairs, keys


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    h, d = case["kv_heads"], case["dim"]
    if case["kind"] == "attend":
        rows = sum(q for _, q in _sequences(case))
        pairs, keys = _pairs(case)
        moved = 2 * rows * case["heads"] * d * size + keys * h * _block_bytes(case)
        return {"bytes": moved + (rows * case["heads"] * 4 if case["lse"] else 0), "flops": 4 * pairs * case["heads"] * d}
    values = 2 * case["tokens"] * h * d
    cache = case["tokens"] * h * _block_bytes(case)
    if case["kind"] == "read":
        return {"bytes": cache + values * size, "flops": values}
    return {"bytes": values * size + 2 * cache + values * 4, "flops": 6 * values}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _inputs(case, seed):
    """The values of a case, from the seed alone: pages in no order, keys with a few strong channels, values without."""
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    cpu = torch.Generator().manual_seed(int(seed))
    dtype, h, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    strong = 1 + 3 * (torch.rand((h, d), generator=gen, device=DEVICE) < 0.04)
    got = {"dtype": dtype}
    if case["kind"] == "attend":
        seqs = _sequences(case)
        need = [-(-n // page) for n, _ in seqs]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=cpu).tolist()
        tables = torch.zeros((len(seqs), max(need)), dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
            at += n
        starts = [0]
        for _, q in seqs:
            starts.append(starts[-1] + q)
        got["q"] = normal(starts[-1], case["heads"], d).to(dtype)
        got["tables"] = tables.to(DEVICE)
        got["lengths"] = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device=DEVICE)
        got["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE) if case["queries"] > 1 else None
        got["prefix"] = None
        if case["prefix"]:
            got["prefix"] = torch.full((len(seqs),), case["prefix"], dtype=torch.int32, device=DEVICE)
        got["slopes"] = None
        if case["slopes"]:
            n = case["heads"]
            got["slopes"] = torch.exp2(-8.0 * torch.arange(1, n + 1, device=DEVICE, dtype=torch.float32) / n)
        got["slots"] = torch.arange(pages * page, device=DEVICE)
    else:
        runs = _runs(case)
        room = [-(-n // page) + 1 for n in runs]  # each stretch may begin in the middle of a page
        pages = sum(room) + 1
        order = torch.randperm(pages, generator=cpu)
        slots, at = [], 0
        for n, p in zip(runs, room):
            first = int(torch.randint(0, page, (1,), generator=cpu))
            place = torch.arange(first, first + n)
            slots.append(order[at : at + p][place // page] * page + place % page)
            at += p
        got["slots"] = torch.cat(slots).to(DEVICE)
    got["pages"] = pages
    got["k"] = (normal(got["slots"].numel(), h, d) * strong).to(dtype)
    got["v"] = normal(got["slots"].numel(), h, d).to(dtype)
    return got


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    fill = case["kind"] != "write"  # a write begins with an empty cache, the others with their tokens in it
    if own:
        from comp_amd import kv

        s["cache"] = kv.KVCache(s["pages"], case["kv_heads"], case["dim"], case["k_format"], case["v_format"], case["page"])
        if fill:
            kv.write(s["cache"], s["k"], s["v"], s["slots"])
    else:
        shape = (s["pages"] * case["page"], case["kv_heads"], case["dim"] // BLOCK)
        s["cache"] = [(torch.zeros((*shape, BLOCK), dtype=torch.int8, device=DEVICE),
                       torch.zeros(shape, dtype=torch.float16, device=DEVICE)) for _ in "kv"]  # fmt: skip
        if fill:
            _plain_write(s)
    if fill:
        del s["k"], s["v"]
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _plain_quantize(x, fmt):
    """f32 [..., 32] -> int8 codes and f16 scales, every step a rounded f32 operation as ggml's formats define it."""
    if fmt == "q8_0":
        d = x.abs().amax(-1)
        d = d / torch.full_like(d, 127.0)  # (a division by a number may be done as a product with its reciprocal)
    else:
        d = x.gather(-1, x.abs().argmax(-1, keepdim=True))[..., 0] / -8.0
    inverse = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    y = x * inverse[..., None]
    if fmt == "q8_0":
        a = y.abs()
        whole = torch.floor(a)
        codes = torch.copysign(torch.where(a - whole >= 0.5, whole + 1, whole), y)
    else:
        codes = torch.clamp(torch.floor(y + 8.5), max=15.0) - 8.0
    return codes.to(torch.int8), d.to(torch.float16)


def _plain_write(s):
    case = s["case"]
    for x, fmt, (codes, scales) in zip((s["k"], s["v"]), (case["k_format"], case["v_format"]), s["cache"]):
        c, d = _plain_quantize(x.float().view(*x.shape[:2], -1, BLOCK), fmt)
        codes[s["slots"]] = c
        scales[s["slots"]] = d


def _plain_values(codes, scales, slots):
    """f32 [..., kv heads, D]: what the codes of these slots stand for."""
    x = codes[slots].float() * scales[slots].float()[..., None]
    return x.flatten(-2)


def _plain_attend(s):
    case, q, lengths = s["case"], s["q"].float(), s["lengths"].long()
    batch, n, h = case["batch"], case["queries"], case["kv_heads"]
    group, page = case["heads"] // h, case["page"]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(batch + 1, device=q.device)
    count = starts[1:] - starts[:-1]
    # queries [batch][n] and keys [batch][length], short sequences padded
    row = torch.arange(n, device=q.device)
    q = q[torch.clamp(starts[:-1, None] + row, max=q.shape[0] - 1)]
    key = torch.arange(case["length"], device=q.device)
    slots = s["tables"].long()[:, key // page] * page + key % page
    k, v = (_plain_values(*half, slots).transpose(1, 2) for half in s["cache"])  # [batch][kv heads][keys][D]
    q = q.view(batch, n, h, group, -1).permute(0, 2, 3, 1, 4).reshape(batch, h, group * n, -1)
    x = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(case["dim"]))
    x = x.view(batch, h, group, n, -1)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    at = (lengths - count)[:, None] + row  # the queries' positions, [batch][n]
    back = at[:, :, None] - key
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, h, group, 1, 1) * back.abs()[:, None, None].float()
    seen = back >= 0
    if s["prefix"] is not None:
        seen |= key < s["prefix"][:, None, None]
    if case["window"]:
        seen &= back < case["window"]
    seen &= key < lengths[:, None, None]
    x = torch.where(seen[:, None, None], x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, h, group * n, -1), v).view(batch, h, group, n, -1)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    # back to the rows that exist: [row][heads][D]
    owner = torch.repeat_interleave(torch.arange(batch, device=q.device), count, output_size=s["q"].shape[0])
    index = torch.arange(s["q"].shape[0], device=q.device) - starts[owner]
    got = [out.permute(0, 3, 1, 2, 4)[owner, index].flatten(1, 2).to(s["dtype"])]
    if case["lse"]:
        lse = (top + torch.log(total))[..., 0]
        got.append(lse.permute(0, 3, 1, 2)[owner, index].flatten(1, 2))
    return got


def _run_own(s):
    from comp_amd import kv

    case = s["case"]
    if case["kind"] == "write":
        kv.write(s["cache"], s["k"], s["v"], s["slots"])
        return kv.read(s["cache"], s["slots"])
    if case["kind"] == "read":
        return kv.read(s["cache"], s["slots"], s["dtype"])
    got = kv.attend(s["cache"], s["q"], s["tables"], s["lengths"], s["starts"], max_queries=case["queries"],
                    softcap=case["softcap"], window=case["window"], prefix=s["prefix"], slopes=s["slopes"],
                    return_lse=case["lse"])  # fmt: skip
    return list(got) if case["lse"] else [got]


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["kind"] == "attend":
        return _plain_attend(s)
    if case["kind"] == "write":
        _plain_write(s)
    dtype = s["dtype"] if case["kind"] == "read" else torch.float32
    return tuple(_plain_values(*half, s["slots"]).to(dtype) for half in s["cache"])


# ---- in 64 bits ------------------------------------------------------------------------------------------------------


def _f32(x):
    return x.to(torch.float32).to(torch.float64)


def _exact_values(x, fmt):
    """f64 [T][kv heads][D]: what the format's definition keeps of x.  Its roundings to f32 and f16 are part of the
    definition; everything between them is in 64 bits (whose quotients and products round to the same f32)."""
    b = x.to(torch.float64).reshape(*x.shape[:2], -1, BLOCK)
    if fmt == "q4_0":
        low, high = b.min(-1).values, b.max(-1).values
        # the value of largest magnitude, the first of them where both signs have it
        place = torch.arange(BLOCK, device=b.device)
        first_low = torch.where(b == low[..., None], place, BLOCK).min(-1).values
        first_high = torch.where(b == high[..., None], place, BLOCK).min(-1).values
        take_high = (high > -low) | ((high == -low) & (first_high < first_low))
        scale = torch.where(take_high, high, low) * -0.125
    else:
        scale = _f32(b.abs().max(-1).values / 127)
    nonzero = scale != 0
    inverse = _f32(torch.where(nonzero, torch.where(nonzero, scale, 1).reciprocal(), 0))
    y = _f32(b * inverse[..., None])
    if fmt == "q4_0":
        code = torch.minimum(torch.floor(_f32(y + 8.5)), torch.tensor(15.0, dtype=torch.float64, device=b.device)) - 8
    else:
        code = torch.sign(y) * torch.floor(y.abs() + 0.5)
    return (code * scale.to(torch.float16).to(torch.float64)[..., None]).flatten(-2)


def exact(case, seed):
    s = _inputs(case, seed)
    k, v = _exact_values(s["k"], case["k_format"]), _exact_values(s["v"], case["v_format"])
    if case["kind"] != "attend":
        return (k, v)
    q = s["q"].to(torch.float64)
    group = case["heads"] // case["kv_heads"]
    out, lse, first = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=q.device), 0
    for b, (n, count) in enumerate(_sequences(case)):
        j = torch.arange(n, device=q.device)
        slots = s["tables"][b].long()[j // case["page"]] * case["page"] + j % case["page"]
        i = torch.arange(n - count, n, device=q.device)[:, None]
        hidden = j > i
        if case["prefix"]:
            hidden = hidden & (j >= case["prefix"])
        if case["window"]:
            hidden = hidden | (j <= i - case["window"])
        for head in range(case["heads"]):
            score = q[first : first + count, head] @ k[slots, head // group].T / case["dim"] ** 0.5
            if case["softcap"]:
                score = torch.tanh(score / case["softcap"]) * case["softcap"]
            if case["slopes"]:
                score = score - s["slopes"][head].double() * (i - j).abs()
            score = score.masked_fill(hidden, -math.inf)
            norm = torch.logsumexp(score, -1)
            empty = norm == -math.inf
            weight = torch.exp(score - norm.masked_fill(empty, 0)[:, None])
            out[first : first + count, head] = weight @ v[slots, head // group]
            lse[first : first + count, head] = norm
        first += count
    return [out, lse] if case["lse"] else [out]
