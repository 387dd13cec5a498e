"""The operators that serving several requests on one decoder is made of, as measurable cases.

Every case is a dict with a "kind":

  sample    the next token of every sequence from its row of logits: temperature, top-k, top-p, min-p, given random numbers
  adapters  low-rank adapters of the tokens' own requests, added to the rows that a shared projection has made
  attend    attention of new rows over a cache that is held in 8 bits, one scale for each block of 64 tokens and head
  store     new rows into that cache, and back as the cache holds them

With `own` false `run` computes the plain form with torch: 32 bits (64 where a choice hangs on a sum), rounded once at the end.
`exact` computes the definitions in 64 bits, in other steps.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 64  # tokens that share a scale
_context = None


def _ctx():
    global _context
    if _context is None:
        from loom_b200 import cabi

        _context = cabi.Context(torch.cuda.current_device())
    return _context


def listed():
    return [
        # one sequence of a small vocabulary, nucleus sampling: the smallest call, all latency
        dict(name="sample 1x32000", kind="sample", rows=1, vocab=32000, mode="nucleus"),
        # a full batch, every request with settings of its own
        dict(name="sample 64x128256", kind="sample", rows=64, vocab=128256, mode="mixed"),
        # one token of one request beside the gate projection of the 2B shape
        dict(name="adapters 1 2560>6912", kind="adapters", tokens=1, cols=2560, rows=6912, slots=8, rank_lo=8, rank_hi=8, order="mixed", dtype="bfloat16"),
        # a step of 16 sequences beside the 8B up-projection, ranks differ, some sequences without an adapter
        dict(name="adapters 16 4096>14336", kind="adapters", tokens=16, cols=4096, rows=14336, slots=12, rank_lo=8, rank_hi=64, order="mixed", dtype="bfloat16"),
        # five requests' prompts in one block of tokens
        dict(name="adapters 2999 2560>6912", kind="adapters", tokens=2999, cols=2560, rows=6912, slots=5, rank_lo=16, rank_hi=16, order="runs", dtype="bfloat16"),
        # float32 adapters of odd sizes, tokens of all requests mixed
        dict(name="adapters f32 333 1000>777", kind="adapters", tokens=333, cols=1000, rows=777, slots=9, rank_lo=3, rank_hi=24, order="mixed", dtype="float32"),
        # one sequence of the 2B shape at context 1040, the smallest attention
        dict(name="attend 1x1040 20/5", kind="attend", seqs=1, length=1039, rows=1, ragged=False, heads=20, kv_heads=5, dim=128),
        # 16 sequences of the 8B shape, ragged, one token each
        dict(name="attend 16x~4000 32/8", kind="attend", seqs=16, length=4000, rows=1, ragged=True, heads=32, kv_heads=8, dim=128),
        # one very long sequence
        dict(name="attend 1x131071 32/8", kind="attend", seqs=1, length=131070, rows=1, ragged=False, heads=32, kv_heads=8, dim=128),
        # the next portion of a long prompt
        dict(name="attend 300 rows at 2900 20/5", kind="attend", seqs=1, length=2900, rows=300, ragged=False, heads=20, kv_heads=5, dim=128),
        # a decode step's rows of 64 sequences
        dict(name="store 64x1 8", kind="store", seqs=64, length=700, rows=1, ragged=True, kv_heads=8, dim=128),
        # eight prompts
        dict(name="store 8x~1000 8", kind="store", seqs=8, length=0, rows=1000, ragged=True, kv_heads=8, dim=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "adapters", "attend", "store"])
    if kind == "sample":
        vocab = _log(rng, 100, 160000)
        return dict(kind=kind, rows=_log(rng, 1, min(256, 64 * 128256 // vocab)), vocab=vocab, mode=rng.choice(["nucleus", "mixed", "topk", "plain"]))
    if kind == "adapters":
        cols, rows = _log(rng, 100, 8000), _log(rng, 100, 15000)
        tokens = _log(rng, 1, min(3000, 28_000_000 // (cols + 2 * rows)))
        lo = rng.randint(1, 32)
        return dict(kind=kind, tokens=tokens, cols=cols, rows=rows, slots=rng.randint(1, 12), rank_lo=lo, rank_hi=rng.randint(lo, 64),
                    order=rng.choice(["mixed", "runs"]), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    kv_heads, dim = rng.randint(1, 8), rng.choice([40, 64, 72, 80, 96, 128, 128, 128, 160, 256])
    if kind == "attend":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        seqs = _log(rng, 1, 32)
        length = _log(rng, 2, 131070 * 8 * 128 // (2 * seqs * kv_heads * dim))
        rows = rng.choice([1, 1, 1, 2, 7, _log(rng, 8, 300)])
        rows = max(1, min(rows, 500_000_000 // (length * heads * seqs)))
        return dict(kind=kind, seqs=seqs, length=length, rows=rows, ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads, dim=dim)
    seqs = _log(rng, 1, 128)
    length = _log(rng, 1, 3000) if rng.random() < 0.6 else 0
    rows = rng.choice([1, 1, rng.randint(2, BLOCK)]) if length else _log(rng, 1, max(2, 8000 // seqs))
    return dict(kind=kind, seqs=seqs, length=length, rows=rows, ragged=rng.random() < 0.7, kv_heads=kv_heads, dim=dim)


# ---- sizes that follow from a case alone -------------------------------------------------------------------------------------


def _shape(case):
    """Positions that every sequence holds before the call, and rows that each one gets."""
    n, length, rows = case["seqs"], case["length"], case["rows"]
    if not case["ragged"]:
        return [length] * n, [rows] * n
    r = random.Random(n * 1000003 + length * 101 + rows)
    lengths = [max(1, int(length * r.uniform(0.3, 1.0))) if length else 0 for _ in range(n)]
    counts = [rows if rows == 1 else max(1, int(rows * r.uniform(0.4, 1.0))) for _ in range(n)]
    if n > 2 and rows > 1:
        counts[1] = 0  # a sequence that takes no part in this call
    return lengths, counts


def _ranks(case):
    r = random.Random(case["slots"] * 7919 + case["rank_lo"] * 31 + case["rank_hi"])
    return [r.randint(case["rank_lo"], case["rank_hi"]) for _ in range(case["slots"])]


def _slots_of_tokens(case):
    r, t, n = random.Random(case["tokens"] * 613 + case["slots"]), case["tokens"], case["slots"]
    if case["order"] == "mixed":
        return [r.randrange(n) if t == 1 or r.random() < 0.9 else -1 for _ in range(t)]
    cuts = sorted(r.randrange(t + 1) for _ in range(n - 1))
    runs = list(range(n))
    r.shuffle(runs)
    return [runs[sum(c <= i for c in cuts)] for i in range(t)]


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return dict(bytes=case["rows"] * (case["vocab"] * 4 + 20 + 8), flops=0)
    if kind == "adapters":
        slots, ranks, size = _slots_of_tokens(case), _ranks(case), 2 if case["dtype"] == "bfloat16" else 4
        cols, rows, t = case["cols"], case["rows"], case["tokens"]
        weights = sum(ranks[s] for s in set(slots) if s >= 0) * (cols + rows) * size
        return dict(bytes=weights + t * (cols + 2 * rows) * 4 + t * 4, flops=2 * (cols + rows) * sum(ranks[s] for s in slots if s >= 0))
    lengths, counts = _shape(case)
    hd = case["kv_heads"] * case["dim"]
    if kind == "store":  # in: the rows, and what is there of a block that they complete; out: codes or rows of the open block; then back
        held = sum((8 if j >= (n + m) // BLOCK * BLOCK else 2) * hd for n, m in zip(lengths, counts) for j in range(n, n + m))
        return dict(bytes=sum(counts) * hd * 16 + 2 * held, flops=0)
    q = case["heads"] * case["dim"]
    seen = sum((n + m) // BLOCK * BLOCK * 2 * hd + (n + m) // BLOCK * 8 * case["kv_heads"] + (n + m) % BLOCK * 8 * hd for n, m in zip(lengths, counts) if m)
    return dict(bytes=seen + sum(counts) * q * 8, flops=4 * q * sum(n + j + 1 for n, m in zip(lengths, counts) for j in range(m)))


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed & 0x7FFFFFFF)
    return g


def _sample_inputs(case, seed):
    g, rows, vocab, mode = _gen(seed), case["rows"], case["vocab"], case["mode"]
    logits = torch.randn(rows, vocab, device="cuda", generator=g) * 2.2
    peaks = torch.randint(0, vocab, (rows, min(24, vocab)), device="cuda", generator=g)
    logits.scatter_add_(1, peaks, torch.rand(peaks.shape, device="cuda", generator=g) * 9.0)
    pick = lambda values, kind: torch.tensor(values, device="cuda", dtype=kind)[torch.randint(0, len(values), (rows,), device="cuda", generator=g)]  # noqa: E731
    temperature, top_k = pick([0.8], torch.float32), pick([0], torch.int32)
    top_p, min_p = pick([1.0], torch.float32), pick([0.0], torch.float32)
    if mode == "nucleus":
        top_p = pick([0.9, 0.95], torch.float32)
    elif mode == "topk":
        top_k = pick([40, 50, 1], torch.int32)
    elif mode == "mixed":
        temperature = pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.3], torch.float32)
        top_k = pick([0, 0, 20, 50, 1000], torch.int32)
        top_p = pick([1.0, 0.8, 0.9, 0.95, 0.99], torch.float32)
        min_p = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
    return dict(logits=logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, uniform=torch.rand(rows, device="cuda", generator=g))


def _adapter_inputs(case, seed):
    g, t, cols, rows, n = _gen(seed), case["tokens"], case["cols"], case["rows"], case["slots"]
    kind = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
    ranks = _ranks(case)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    return dict(x=randn(t, cols), base=randn(t, rows), slot=torch.tensor(_slots_of_tokens(case), device="cuda", dtype=torch.int32),
                down=[(randn(r, cols) / math.sqrt(cols)).to(kind) for r in ranks], up=[(randn(rows, r) * 0.3 / math.sqrt(r)).to(kind) for r in ranks],
                scale=torch.rand(n, device="cuda", generator=g) * 2 + 0.5, ranks=ranks)


def _kv_inputs(case, seed, rows):
    """`rows` rows of keys and values: channels of different spread, as keys have them."""
    g, h, d = _gen(seed), case["kv_heads"], case["dim"]
    spread = torch.exp(torch.randn(h, d, device="cuda", generator=g) * 0.5)
    k = torch.randn(rows, h, d, device="cuda", generator=g) * spread
    v = torch.randn(rows, h, d, device="cuda", generator=g)
    return k, v, g


def _starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), device="cuda", dtype=torch.int32)


def _attend_inputs(case, seed):
    lengths, counts = _shape(case)
    whole = [n + m if m else 0 for n, m in zip(lengths, counts)]
    k, v, g = _kv_inputs(case, seed, sum(whole))
    q = torch.randn(sum(counts), case["heads"], case["dim"], device="cuda", generator=g) * 1.2
    return lengths, counts, whole, k, v, q


# ---- the plain form's cache: [sequence, position, head, dim] padded, codes and scales of whole blocks, the open block as it is ---


def _round(r):
    return torch.sign(r) * torch.floor(torch.abs(r) + 0.5)


def _quantize(blocks):
    """Blocks [..., 64, heads, dim] of float32 rows: codes and each block's and head's largest value."""
    amax = blocks.abs().amax(dim=(-3, -1))
    wide = amax.double()
    s = torch.where(wide > 0, torch.full_like(wide, 127.0) / wide, torch.zeros_like(wide))
    return _round(blocks.double() * s[..., None, :, None]).clamp(-128, 127).to(torch.int8), amax


def _dequantize(codes, amax):
    return codes.float() * (amax / torch.full_like(amax, 127.0))[..., None, :, None]


def _padded(rows, counts, at, length):
    """Rows of all sequences, one behind the other, as [sequence, length, ...], sequence i's from place at[i] on."""
    n, device = len(counts), rows.device
    out = torch.zeros((n, length) + tuple(rows.shape[1:]), device=device)
    count = torch.tensor(counts, device=device)
    seq = torch.repeat_interleave(torch.arange(n, device=device), count)
    place = torch.arange(rows.shape[0], device=device) - (torch.cumsum(count, 0) - count)[seq] + torch.tensor(at, device=device)[seq]
    out[seq, place] = rows
    return out


def _plain_cache(rows, counts):
    whole = -(-max(max(counts), 1) // BLOCK) * BLOCK
    blocks = _padded(rows, counts, [0] * len(counts), whole).unflatten(1, (-1, BLOCK))
    codes, amax = _quantize(blocks)
    n = torch.tensor(counts, device=rows.device)
    i = torch.arange(len(counts), device=rows.device)
    last = torch.clamp(n // BLOCK, max=blocks.shape[1] - 1)
    return codes, amax, blocks[i, last].clone()


def prepare(case, seed):
    kind = case["kind"]
    if kind == "sample":
        s = _sample_inputs(case, seed)
        s.update(kind=kind, tokens=torch.empty(case["rows"], device="cuda", dtype=torch.int32), logprob=torch.empty(case["rows"], device="cuda"))
        return s
    if kind == "adapters":
        s = _adapter_inputs(case, seed)
        t, cols, rows, n, ranks = case["tokens"], case["cols"], case["rows"], case["slots"], s["ranks"]
        s.update(kind=kind, out=torch.empty(t, rows, device="cuda"))
        if own:
            from loom_b200 import cabi

            code = cabi.DTYPES[case["dtype"]]
            s["adapters"] = cabi.Adapters(_ctx(), n, rows, cols, max(ranks), code)
            torch.cuda.synchronize()
            for i in range(n):
                s["adapters"].put(i, s["down"][i], s["up"][i], float(s["scale"][i]), code)
            _ctx().sync()
        else:
            most = max(ranks)
            s["downs"] = torch.zeros(n, most, cols, device="cuda", dtype=s["down"][0].dtype)
            s["ups"] = torch.zeros(rows, n, most, device="cuda", dtype=s["up"][0].dtype)
            for i, r in enumerate(ranks):
                s["downs"][i, :r] = s["down"][i]
                s["ups"][:, i, :r] = s["up"][i]
        del s["down"], s["up"]
        return s
    lengths, counts = _shape(case)
    rows, h, d = sum(counts), case["kv_heads"], case["dim"]
    s = dict(kind=kind, rows=rows, heads=case.get("heads"), starts=_starts(counts), lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32), most=max(counts))
    longest = max(n + m for n, m in zip(lengths, counts))
    if kind == "attend":
        _, _, whole, k, v, s["q"] = _attend_inputs(case, seed)
        s["out"] = torch.empty_like(s["q"])
        if own:
            s["cache"] = _filled(case, longest, whole, k, v)
        else:
            s["k"], s["v"] = _plain_cache(k, whole), _plain_cache(v, whole)
            s["whole"] = torch.tensor(whole, device="cuda")
        return s
    # what the sequences' open blocks hold already, then the new rows
    open_ = [n % BLOCK for n in lengths]
    k, v, _ = _kv_inputs(case, seed, sum(open_) + rows)
    s["new_k"], s["new_v"] = k[sum(open_):].contiguous(), v[sum(open_):].contiguous()
    s["out_k"], s["out_v"] = torch.empty_like(s["new_k"]), torch.empty_like(s["new_v"])
    old_k, old_v = k[: sum(open_)], v[: sum(open_)]
    if own:
        s["cache"] = _filled(case, longest, open_, old_k, old_v, [n // BLOCK * BLOCK for n in lengths])
    else:
        s["old_k"], s["old_v"], s["counts"] = _padded(old_k, open_, [0] * len(open_), BLOCK), _padded(old_v, open_, [0] * len(open_), BLOCK), torch.tensor(counts, device="cuda")
    return s


def _filled(case, longest, counts, k, v, at=None):
    from loom_b200 import cabi

    cache = cabi.KV8(_ctx(), case["seqs"], longest, case["kv_heads"], case["dim"])
    starts, lengths = _starts(counts), torch.tensor(at or [0] * len(counts), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    if sum(counts):
        cache.append(sum(counts), lengths, k, v, starts=starts)
        _ctx().sync()
    return cache


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def run(s):
    kind = s["kind"]
    if own:
        if kind == "sample":
            _ctx().sample(s["logits"].shape[0], s["logits"].shape[1], s["logits"], s["uniform"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"], logprob=s["logprob"])
            return s["tokens"], s["logprob"]
        if kind == "adapters":
            s["adapters"].apply(s["x"].shape[0], s["slot"], s["x"], s["out"], base=s["base"])
            return s["out"]
        if kind == "attend":
            s["cache"].attend(s["rows"], s["heads"], s["lengths"], s["q"], s["out"], starts=s["starts"])
            return s["out"]
        s["cache"].append(s["rows"], s["lengths"], s["new_k"], s["new_v"], starts=s["starts"])
        s["cache"].read(s["rows"], s["lengths"], s["out_k"], s["out_v"], starts=s["starts"])
        return s["out_k"], s["out_v"]
    return {"sample": _sample_plain, "adapters": _adapters_plain, "attend": _attend_plain, "store": _store_plain}[kind](s)


def _sample_plain(s):
    logits, u = s["logits"], s["uniform"].double()[:, None]
    vocab = logits.shape[1]
    temperature = s["temperature"].double()[:, None]
    greedy = ~(temperature > 0)
    wide = logits.double()
    top = wide.amax(1, keepdim=True)
    w = torch.exp((wide - top) / torch.where(greedy, 1.0, temperature))
    place = torch.sort(logits, dim=1, descending=True, stable=True).indices
    rank = torch.arange(vocab, device=logits.device)[None]
    ordered = w.gather(1, place)
    k = s["top_k"].long()[:, None]
    keep = rank < torch.where(k > 0, k, vocab)
    mass = torch.cumsum(ordered * keep, 1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (before < p * mass[:, -1:]) | (rank == 0)
    keep &= ordered >= s["min_p"].double()[:, None]
    keep = torch.where(greedy, rank == 0, keep)
    kept = torch.zeros_like(w).scatter(1, place, ordered * keep)
    cdf = torch.cumsum(kept, 1)
    total = cdf[:, -1:]
    token = (cdf <= u * total).sum(1, keepdim=True)
    return token[:, 0].int(), torch.log(w.gather(1, token) / total)[:, 0].float()


def _adapters_plain(s):
    n, most, cols = s["downs"].shape
    x = s["x"]
    h = (x @ s["downs"].reshape(n * most, cols).float().T).unflatten(1, (n, most))
    mine = (s["slot"][:, None] == torch.arange(n, device=x.device)[None]).float() * s["scale"][None]
    return s["base"] + (h * mine[..., None]).flatten(1) @ s["ups"].flatten(1).float().T


def _plain_rows(cache, whole):
    codes, amax, last = cache
    rows = _dequantize(codes, amax).flatten(1, 2)
    i = torch.arange(len(whole), device=rows.device)[:, None]
    at = torch.clamp(whole // BLOCK, max=codes.shape[1] - 1)[:, None] * BLOCK + torch.arange(BLOCK, device=rows.device)[None]
    is_open = at >= (whole // BLOCK * BLOCK)[:, None]
    rows[i, at] = torch.where(is_open[..., None, None], last, rows[i, at])
    return rows


def _attend_plain(s):
    q, starts, lengths = s["q"], s["starts"].long(), s["lengths"].long()
    k, v = _plain_rows(s["k"], s["whole"]), _plain_rows(s["v"], s["whole"])
    n, length, h, d = k.shape
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.bucketize(row, starts[1:], right=True)
    j = row - starts[seq]
    wide = torch.zeros(n, s["most"], h, q.shape[1] // h, d, device=q.device)
    wide[seq, j] = q.unflatten(1, (h, -1))
    scores = torch.einsum("smhgd,slhd->shgml", wide, k) / math.sqrt(d)
    seen = torch.arange(length, device=q.device)[None, None] <= lengths[:, None, None] + torch.arange(s["most"], device=q.device)[None, :, None]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.einsum("shgml,slhd->smhgd", p / p.sum(-1, keepdim=True), v)
    return out[seq, j].flatten(1, 2)


def _store_plain(s):
    starts, lengths, counts = s["starts"].long(), s["lengths"].long(), s["counts"]
    n, device = len(counts), starts.device
    row = torch.arange(s["rows"], device=device)
    seq = torch.bucketize(row, starts[1:], right=True)
    at = row - starts[seq] + lengths[seq] % BLOCK  # counted from the open block's first position
    space = -(-(BLOCK + s["most"]) // BLOCK)
    closed = at < ((lengths % BLOCK + counts) // BLOCK * BLOCK)[seq]

    def one(old, new):
        rows = torch.zeros((n, space * BLOCK) + tuple(new.shape[1:]), device=device)
        rows[:, :BLOCK] = old
        rows[seq, at] = new
        back = _dequantize(*_quantize(rows.unflatten(1, (space, BLOCK)))).flatten(1, 2)
        return torch.where(closed[:, None, None], back[seq, at], new)

    return one(s["old_k"], s["new_k"]), one(s["old_v"], s["new_v"])


# ---- the definitions in 64 bits, sequence by sequence ------------------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return {"sample": _sample_exact, "adapters": _adapters_exact, "attend": _attend_exact, "store": _store_exact}[case["kind"]](case, seed)


def _sample_exact(case, seed):
    s = {k: v.cpu().numpy() for k, v in _sample_inputs(case, seed).items()}
    tokens, logprob = [], []
    for i in range(case["rows"]):
        row, t = s["logits"][i].astype(np.float64), float(s["temperature"][i])
        if not t > 0:
            tokens.append(int(np.argmax(row)))
            logprob.append(0.0)
            continue
        order = np.lexsort((np.arange(row.size), -row))
        w = np.exp((row[order] - row[order[0]]) / t)
        if 0 < s["top_k"][i] < row.size:
            order, w = order[: s["top_k"][i]], w[: s["top_k"][i]]
        p = float(s["top_p"][i])
        if p < 1:
            mass = np.cumsum(w.astype(np.longdouble))
            n = int(np.searchsorted(mass, p * mass[-1], side="left")) + 1
            order, w = order[:n], w[:n]
        fine = w >= float(s["min_p"][i])
        order, w = order[fine], w[fine]
        by_index = np.argsort(order, kind="stable")
        mass = np.cumsum(w[by_index].astype(np.longdouble))
        at = by_index[int(np.searchsorted(mass, float(s["uniform"][i]) * mass[-1], side="right"))]
        tokens.append(int(order[at]))
        logprob.append(float(np.log(w[at] / mass[-1])))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprob, dtype=torch.float64)


def _adapters_exact(case, seed):
    s = _adapter_inputs(case, seed)
    out = s["base"].double()
    for i in range(case["slots"]):
        mine = s["slot"] == i
        if bool(mine.any()):
            out[mine] += float(s["scale"][i]) * (s["x"][mine].double() @ s["down"][i].double().T) @ s["up"][i].double().T
    return out


def _held(rows, whole):
    """Rows [positions, dim] of one sequence and head, in 64 bits, as the cache holds them."""
    rows, closed = rows.double(), whole // BLOCK * BLOCK
    if not closed:
        return rows
    blocks = rows[:closed].reshape(-1, BLOCK, rows.shape[-1])
    top = blocks.abs().flatten(1).max(1).values[:, None, None]
    step = 127.0 * torch.where(top > 0, 1 / top, 0.0)
    near = torch.round(blocks * step)
    # (a reciprocal and a product are not the quotient: values next to the middle of two codes go by the quotient itself)
    tie = (blocks * step - torch.floor(blocks * step) - 0.5).abs() < 1e-9
    r = blocks * (torch.full_like(top, 127.0) / torch.where(top > 0, top, 1.0))
    codes = torch.where(tie, torch.copysign(torch.floor(r.abs() + 0.5), r), near)
    return torch.cat([(codes * top / 127.0).reshape(closed, -1), rows[closed:whole]])


def _attend_exact(case, seed):
    lengths, counts, whole, k, v, q = _attend_inputs(case, seed)
    h, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out, at, row = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0, 0
    for n, m, w in zip(lengths, counts, whole):
        for i in range(h if m else 0):
            kk, vv = _held(k[at:at + w, i], w), _held(v[at:at + w, i], w)
            scores = torch.tensordot(q[row:row + m, i * group:(i + 1) * group].double(), kk, dims=([2], [1])) / math.sqrt(case["dim"])
            late = torch.arange(w, device="cuda")[None] > n + torch.arange(m, device="cuda")[:, None]
            scores[late[:, None].expand(scores.shape)] = float("-inf")
            out[row:row + m, i * group:(i + 1) * group] = torch.softmax(scores, -1) @ vv
        at, row = at + w, row + m
    return out


def _store_exact(case, seed):
    lengths, counts = _shape(case)
    open_ = [n % BLOCK for n in lengths]
    k, v, _ = _kv_inputs(case, seed, sum(open_) + sum(counts))
    got = []
    for rows in (k, v):
        out, at, row = torch.empty(sum(counts), case["kv_heads"], case["dim"], dtype=torch.float64, device="cuda"), 0, 0
        for o, m in zip(open_, counts):
            both = torch.cat([rows[at:at + o], rows[sum(open_) + row:sum(open_) + row + m]])
            for i in range(case["kv_heads"] if m else 0):
                out[row:row + m, i] = _held(both[:, i], o + m)[o:]
            at, row = at + o, row + m
        got.append(out)
    return tuple(got)
