"""The paged key-value cache: what is measured of its three operators.

write   new tokens' keys and values are quantised into the pages of their sequences and read back as stored
read    cached tokens are read back as the values that their codes stand for
attend  one new token a sequence attends over its cached keys and values

Formats of the cache: "f16" and "bf16" hold the rounded values; "mx8" holds e4m3 codes and "mx4" e2m1 codes, both
with one power-of-two scale for every 32 consecutive elements of a head's vector: the smallest 2^e, e >= -126, with
max|x| <= 448 * 2^e (mx8) or 6 * 2^e (mx4); codes are x / 2^e rounded to nearest, ties to even.
"""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # --- one new token a sequence over the cache
        # a single conversation at its beginning: latency is everything
        dict(name="attend_one_short", op="attend", format="f16", type="f16", batch=1, kv_heads=8, group=4, dim=128, page=16,
             shortest=127, tokens=127, window=0),
        # 12 heads of 64 (the encoder's own head layout), no shared heads, 32-bit activations, ragged, pages of 48
        dict(name="attend_heads_of_64_f32", op="attend", format="f16", type="f32", batch=128, kv_heads=12, group=1, dim=64,
             page=48, shortest=0, tokens=511, window=0),
        # a serving batch of mixed lengths, one of them empty
        dict(name="attend_batch_mx8", op="attend", format="mx8", type="bf16", batch=64, kv_heads=8, group=4, dim=128, page=32,
             shortest=0, tokens=4097, window=0),
        # one long document
        dict(name="attend_long_mx8", op="attend", format="mx8", type="f16", batch=1, kv_heads=8, group=4, dim=128, page=64,
             shortest=131071, tokens=131071, window=0),
        # the same question over 4-bit pages, a batch of long documents
        dict(name="attend_long_batch_mx4", op="attend", format="mx4", type="bf16", batch=16, kv_heads=8, group=8, dim=128,
             page=64, shortest=4000, tokens=32768, window=0),
        # all query heads share one key head of 256, only the last 1,024 positions are seen
        dict(name="attend_one_kv_head_window", op="attend", format="bf16", type="bf16", batch=96, kv_heads=1, group=16, dim=256,
             page=16, shortest=500, tokens=6000, window=1024),
        # the largest: a full batch over 16-bit pages
        dict(name="attend_batch_f16", op="attend", format="f16", type="f16", batch=32, kv_heads=8, group=8, dim=128, page=128,
             shortest=8192, tokens=8192, window=0),
        # --- quantised as it is written
        # one token for each sequence of a serving batch
        dict(name="write_one_token_mx8", op="write", format="mx8", type="bf16", batch=64, kv_heads=8, dim=128, page=32,
             shortest=1, tokens=1, start=1500),
        # prompts of mixed lengths, continued in the middle of a page
        dict(name="write_prompts_mx8", op="write", format="mx8", type="f16", batch=9, kv_heads=8, dim=128, page=64, shortest=1,
             tokens=16384, start=37),
        # long prompts to 4 bits from 32-bit activations, heads of 96
        dict(name="write_prompts_mx4_f32", op="write", format="mx4", type="f32", batch=5, kv_heads=4, dim=96, page=16,
             shortest=100, tokens=20001, start=0),
        # --- read back
        # a short prefix for one sequence
        dict(name="read_prefix_mx4", op="read", format="mx4", type="f16", batch=1, kv_heads=8, dim=128, page=16, shortest=333,
             tokens=333, start=0),
        # whole documents, as they are handed to a prompt's attention
        dict(name="read_documents_mx8", op="read", format="mx8", type="bf16", batch=8, kv_heads=8, dim=128, page=64,
             shortest=1000, tokens=16384, start=5),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    c = dict(op=rng.choice(["attend", "attend", "write", "read"]), format=rng.choice(["f16", "bf16", "mx8", "mx4"]),
             type=rng.choice(["f32", "f16", "bf16"]), dim=rng.choice([32, 64, 96, 128, 192, 256]),
             kv_heads=rng.choice([1, 2, 3, 4, 8, 12]), page=rng.choice([16, 32, 48, 64, 128, 256]), batch=log(1, 128))
    per_token = c["kv_heads"] * c["dim"]
    if c["op"] == "attend":
        c["group"] = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16, 32])
        # no more than a third of the largest listed case's cached elements and of its scores
        most = min(32 * 8192 * 1024 // (c["batch"] * per_token), 32 * 8192 * 64 // (c["batch"] * c["kv_heads"] * c["group"])) // 3
        c["tokens"] = log(1, max(2, min(most, 60000)))
        c["window"] = rng.choice([0, 0, 0, 128, 1000])
    else:
        c["tokens"] = log(1, max(2, min(16384 * 4 * 1024 // (c["batch"] * per_token), 20000)))
        c["start"] = rng.choice([0, rng.randrange(1, 2000)])
    c["shortest"] = rng.choice([0, 1, c["tokens"] // 2, c["tokens"]])
    return c


def _counts(case):
    """Tokens of each sequence: the first the longest, the second the shortest, the others spread between."""
    lo, hi, n = case["shortest"], case["tokens"], case["batch"]
    c = [lo + (i * 2654435761 + 97) % 4294967296 * (hi - lo + 1) // 4294967296 for i in range(n)]
    c[0] = hi
    if n > 1:
        c[1] = lo
    return c


def _inputs(case, seed):
    """Everything that a case holds, from the seed: keys, values and queries as a model's projections give them."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    counts = _counts(case)
    total, start = sum(counts), case.get("start", 0)
    t, h, d, page = TYPES[case["type"]], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # keys: a few channels of each head are large in every token; values: no such channels, tokens of unlike size
    loud = 1 + 7 * (torch.rand((h, d), generator=g, device="cuda") < 0.04)
    x = {"key": normal(total, h, d).mul_(loud).to(t),
         "value": normal(total, h, d).mul_(torch.exp2(normal(total, h, 1))).to(t)}
    if case["op"] == "attend":
        x["query"] = normal(case["batch"], h * case["group"], d).to(t)
    per = [-(-(start + n) // page) for n in counts]
    width, pages = max(1, max(per)), sum(per) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.tensor(per, device="cuda")[:, None]
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    table[used] = order[:sum(per)]
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    cu = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
    cu[1:] = n.cumsum(0)
    x |= {"pages": pages, "table": table, "counts": n, "cu": cu, "starts": torch.full_like(n, start), "total": total}
    return x


def _slots(x, page):
    """The flat place of every new token in the pages."""
    seq = torch.repeat_interleave(x["counts"].long(), output_size=x["total"])
    pos = torch.arange(x["total"], device="cuda") - x["cu"].long()[seq] + x["starts"].long()[seq]
    return x["table"].long()[seq, pos // page] * page + pos % page


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, **x}
    if own:
        import eos_b200
        s["runtime"] = _runtime()
        s["cache"] = eos_b200.KvCache(s["runtime"], x["pages"], case["page"], case["kv_heads"], case["dim"], case["format"])
        if case["op"] != "write":
            _own_append(s)
            torch.cuda.synchronize()
    else:
        h, d, n = case["kv_heads"], case["dim"], x["pages"] * case["page"]
        codes = {"f16": torch.float16, "bf16": torch.bfloat16, "mx8": torch.float8_e4m3fn, "mx4": torch.uint8}[case["format"]]
        for name in ("key", "value"):
            s[name + "_codes"] = torch.zeros((n, h, d // 2 if case["format"] == "mx4" else d), dtype=torch.uint8, device="cuda") \
                if case["format"][:2] == "mx" else torch.zeros((n, h, d), dtype=codes, device="cuda")
            s[name + "_scales"] = torch.ones((n, h, d // 32), dtype=torch.uint8, device="cuda")
        s["slots"] = _slots(x, case["page"])
        if case["op"] != "write":
            _plain_write(s)
    if case["op"] != "write":
        del s["key"], s["value"]
    return s


_kept = []


def _runtime():
    if not _kept:
        import eos_b200
        _kept.append(eos_b200.Runtime(torch.cuda.current_device()))
    return _kept[0]


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "attend":
            return _own_attend(state)
        if op == "write":
            _own_append(state)
        return _own_read(state)
    if op == "attend":
        return _plain_attend(state)
    if op == "write":
        _plain_write(state)
    return _plain_read(state)


# ------------------------------------------------------------------------------------------- the framework's calls

def _own_append(s):
    c = s["case"]
    s["cache"].append_device(s["key"].data_ptr(), s["value"].data_ptr(), c["type"], s["total"], c["batch"],
                             s["table"].data_ptr(), s["table"].shape[1], s["starts"].data_ptr(), s["cu"].data_ptr(),
                             stream=torch.cuda.current_stream().cuda_stream)


def _own_read(s):
    c = s["case"]
    k = torch.empty((s["total"], c["kv_heads"], c["dim"]), dtype=TYPES[c["type"]], device="cuda")
    v = torch.empty_like(k)
    s["cache"].read_device(k.data_ptr(), v.data_ptr(), c["type"], s["total"], c["batch"], s["table"].data_ptr(),
                           s["table"].shape[1], s["starts"].data_ptr(), s["cu"].data_ptr(),
                           stream=torch.cuda.current_stream().cuda_stream)
    return [k, v]


def _own_attend(s):
    c, q = s["case"], s["query"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    s["cache"].attend_device(q.data_ptr(), c["type"], q.shape[1], c["batch"], s["table"].data_ptr(), s["table"].shape[1],
                             s["counts"].data_ptr(), out.data_ptr(), scale=c["dim"] ** -0.5, window=c["window"],
                             d_lse=lse.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return [out, lse]


# ------------------------------------------------------------------------------------------------ the plain forms

def _scales_of(x, limit):
    """Biased exponents of the blocks' scales from 32-bit values [..., blocks, 32]; limit: mantissa bits of the type's
    largest value and its exponent."""
    bits = x.abs().amax(-1).view(torch.int32)
    return torch.clamp((bits >> 23) - limit[1] + ((bits & 0x7FFFFF) > limit[0]).to(torch.int32), min=1)


def _power(e):
    """2^(e - 127) for 1 <= e <= 253."""
    return (e << 23).view(torch.float32)


def _plain_write(s):
    f = s["case"]["format"]
    for name in ("key", "value"):
        x, codes = s[name].float(), s[name + "_codes"]
        if f in ("f16", "bf16"):
            codes[s["slots"]] = x.to(codes.dtype)
            continue
        b = x.view(*x.shape[:-1], -1, 32)
        e = _scales_of(b, (0x600000, 8) if f == "mx8" else (0x400000, 2))
        y = b * _power(254 - e)[..., None]
        s[name + "_scales"][s["slots"]] = e.to(torch.uint8)
        if f == "mx8":
            codes[s["slots"]] = y.to(torch.float8_e4m3fn).view(torch.uint8).view(x.shape)
        else:
            a = y.abs()
            n = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, 2 + torch.round(a), 4 + torch.round(a / 2)))
            n = (n.to(torch.uint8) + 8 * (y < 0).to(torch.uint8)).view(x.shape)
            codes[s["slots"]] = n[..., 0::2] + 16 * n[..., 1::2]


def _plain_values(s, name, at):
    """The 32-bit values of the cached vectors at the places `at`."""
    f, c = s["case"]["format"], s[name + "_codes"][at]
    if f in ("f16", "bf16"):
        return c.float()
    if f == "mx8":
        y = c.view(torch.float8_e4m3fn).float()
    else:
        y = torch.stack([c & 15, c >> 4], -1).flatten(-2).long()
        y = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")[y]
    e = s[name + "_scales"][at].to(torch.int32)
    return (y.view(*y.shape[:-1], -1, 32) * _power(e)[..., None]).flatten(-2)


def _plain_read(s):
    t = TYPES[s["case"]["type"]]
    return [_plain_values(s, "key", s["slots"]).to(t), _plain_values(s, "value", s["slots"]).to(t)]


def _plain_attend(s):
    c, q, page = s["case"], s["query"].float(), s["case"]["page"]
    at = (s["table"].long().clamp(min=0)[:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)
    pos, n = torch.arange(at.shape[1], device="cuda")[None], s["counts"].long()[:, None]
    seen = pos < n
    if c["window"]:
        seen &= pos >= n - c["window"]
    k = _plain_values(s, "key", at).permute(0, 2, 3, 1)
    x = torch.matmul(q.view(c["batch"], c["kv_heads"], c["group"], c["dim"]), k) * c["dim"] ** -0.5
    del k
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    v = _plain_values(s, "value", at).permute(0, 2, 1, 3)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    return [out.view(q.shape).to(s["query"].dtype), (m + torch.log(total)).view(q.shape[:2])]


# ------------------------------------------------------------------------------------------------ cost and definition

def work(case):
    counts, h, d = _counts(case), case["kv_heads"], case["dim"]
    vector = {"f16": 2 * d, "bf16": 2 * d, "mx8": d + d // 32, "mx4": d // 2 + d // 32}[case["format"]]
    wide = 4 if case["type"] == "f32" else 2
    if case["op"] == "attend":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in counts)
        rows = case["batch"] * h * case["group"]
        return {"bytes": 2 * seen * h * vector + rows * (2 * d * wide + 4), "flops": 4 * seen * h * case["group"] * d}
    # a write reads the new vectors, stores their codes, reads the codes and gives the values
    moved = 2 * sum(counts) * h
    return {"bytes": moved * (2 * (d * wide + vector) if case["op"] == "write" else d * wide + vector), "flops": moved * d}


def _stored(x, fmt):
    """The values that the cache holds for `x`, in 64 bits, from the formats' definition."""
    if fmt in ("f16", "bf16"):
        return x.double().to(TYPES[fmt]).double() if fmt == "f16" else x.bfloat16().double()
    b = x.double().unflatten(-1, (-1, 32))
    # largest value 0.875 * 2^9 with 3 mantissa bits down to 2^-6, or 0.75 * 2^3 with one bit down to 2^0
    top, over, mantissa, least = (0.875, 9, 3, -6) if fmt == "mx8" else (0.75, 3, 1, 0)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, e - over + (m > top).to(e.dtype), -126).clamp(min=-126)
    y = torch.ldexp(b, -e)
    _, place = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(place - 1, min=least) - mantissa)
    return torch.ldexp(torch.round(y / step) * step, e).flatten(-2)


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] != "attend":
        return [_stored(x["key"], case["format"]), _stored(x["value"], case["format"])]
    d, g, counts = case["dim"], case["group"], _counts(case)
    out = torch.zeros(x["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(x["query"].shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    end = 0
    for i, n in enumerate(counts):
        end += n
        lo = end - (min(n, case["window"]) if case["window"] else n)
        if lo == end:
            continue
        k, v = (_stored(x[name][lo:end], case["format"]) for name in ("key", "value"))
        q = x["query"][i].double().view(-1, g, d)
        z = torch.einsum("hgd,lhd->hgl", q, k) / d ** 0.5
        lse[i] = torch.logsumexp(z, -1).flatten()
        out[i] = torch.einsum("hgl,lhd->hgd", torch.softmax(z, -1), v).reshape(-1, d)
    return [out, lse]
