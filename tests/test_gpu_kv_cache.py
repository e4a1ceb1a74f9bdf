"""Paged key-value cache on the device: what is stored (exactly), what is read back, and the attention over it, against
a plain implementation in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def stored(x, fmt):
    """What the cache holds for x ([..., dim], any float type), as float64: blocks of 32, the smallest power-of-two scale
    >= 2^-126 under which the type's largest value is not passed, round to nearest even."""
    if fmt in ("f16", "bf16"):
        return x.float().to(DTYPES[fmt]).double()
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top, mant, low = (448.0, 3, -6) if fmt == "mx8" else (6.0, 1, 0)
    amax = b.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    amax = torch.where(bad, torch.zeros_like(amax), amax)
    e = torch.where(amax > 0, torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / top)), torch.full_like(amax, -126.0))
    for _ in range(2):   # log2 may be off by a rounding
        e = torch.where(amax > top * torch.exp2(e), e + 1, e)
        e = torch.where(amax <= top * torch.exp2(e - 1), e - 1, e)
    e = e.clamp(min=-126)
    y = torch.where(bad, torch.zeros_like(b), b) * torch.exp2(-e)
    place = torch.floor(torch.log2(torch.where(y == 0, torch.ones_like(y), y.abs())))
    step = torch.exp2(torch.clamp(place, min=low) - mant)
    r = torch.round(y / step) * step * torch.exp2(e)
    return torch.where(bad, torch.full_like(r, float("nan")), r).reshape(x.shape)


class Sequences:
    """Page tables of ragged sequences in a cache, pages in random order, entries behind a sequence's end out of range."""

    def __init__(self, fmt, dim, heads, page, capacity, seed=0, spare=2, runtime=None):
        import eos_b200
        rng = np.random.default_rng(seed)
        per = [-(-c // page) for c in capacity]
        self.pages = sum(per) + spare
        order = rng.permutation(self.pages)
        self.max_pages = max(1, max(per)) + 1
        table = np.full((len(capacity), self.max_pages), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = torch.from_numpy(table).cuda()
        self.rt = runtime or eos_b200.Runtime(0)
        self.cache = eos_b200.KvCache(self.rt, self.pages, page, heads, dim, fmt)
        self.batch, self.heads, self.dim, self.fmt, self.page = len(capacity), heads, dim, fmt, page

    def _ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def append(self, k, v, starts, counts=None, strides=None, type_=None, tokens=None):
        cu = None if counts is None else self._ints([0] + list(np.cumsum(counts)))
        st = self._ints(starts)
        name = type_ or {d: n for n, d in DTYPES.items()}[k.dtype]
        self.cache.append_device(k.data_ptr(), v.data_ptr(), name, k.shape[0] if tokens is None else tokens, self.batch,
                                 self.table.data_ptr(), self.max_pages, st.data_ptr(), None if cu is None else cu.data_ptr(),
                                 strides, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()

    def read(self, starts, counts, type_="f32", fill=None):
        n = sum(counts)
        extra = 0 if fill is None else 5
        k = torch.full((n + extra, self.heads, self.dim), 0.0 if fill is None else fill, dtype=DTYPES[type_], device="cuda")
        v = k.clone()
        cu, st = self._ints([0] + list(np.cumsum(counts))), self._ints(starts)
        self.cache.read_device(k.data_ptr(), v.data_ptr(), type_, n + extra, self.batch, self.table.data_ptr(), self.max_pages,
                               st.data_ptr(), cu.data_ptr(), None, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return k, v

    def attend(self, q, lengths, scale, window=0, query_strides=(0, 0), type_=None, shape=None, stream=None):
        n = self._ints(lengths)
        shape = shape or q.shape
        out = torch.full(shape, 7.0, dtype=q.dtype, device="cuda")
        lse = torch.full(shape[:2], 7.0, device="cuda")
        name = type_ or {d: n_ for n_, d in DTYPES.items()}[q.dtype]
        torch.cuda.synchronize()
        self.cache.attend_device(q.data_ptr(), name, shape[1], self.batch, self.table.data_ptr(), self.max_pages, n.data_ptr(),
                                 out.data_ptr(), scale, window, lse.data_ptr(), query_strides,
                                 torch.cuda.current_stream().cuda_stream if stream is None else stream)
        torch.cuda.synchronize()
        return out, lse

    def sync(self):
        self.cache.sync(torch.cuda.current_stream().cuda_stream)


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def check_attend(q, kv, lengths, scale, window, fmt, out, lse, group):
    """Elementwise, against 64 bits over the stored values.  With S = scale sum |q k| and u = 2^-23 (a sum in the tensor
    core may be cut rather than rounded) a score is off by at most
        d = S (2 split + (dim + 8) u),  split = 2^-22 (f16 operands: 11 + 11 bits) or 2^-16 (bf16: 8 + 8),
    a weight by the factor 2 d + 2^-20 (exp2, and its argument's rounding), and n weighted values add n u and the
    weights' split; the result is rounded once more to its type.  Numerator and denominator each carry this once.
    Weights of bf16 results are one f16 number (unless the cache is bf16), in the numerator alone: half a step, 2^-11.
    Below f16's normal numbers a split factor is off by 2^-25 absolutely instead.  Query rows are scaled to a largest
    magnitude of at least 2^13, so that is 2^-38 of it.  Weights, times their value's scale s_j, are scaled to a largest of
    at least 2^6, so that is 2^-31 max(p s): 2^-31 sum_j |v_j| for f16 (s = 1); for the block-scaled formats s_j is at most
    max|v_j| 2 / 28672 and the codes |v_j| / s_j are at most 49152, together n 2^-29 max_j(p_j max|v_j|)."""
    split = 2.0 ** -16 if fmt == "bf16" else 2.0 ** -22
    u = 2.0 ** -23
    half = HALF_STEP[{d: n for n, d in DTYPES.items()}[out.dtype]]
    for b, n in enumerate(lengths):
        lo = max(0, n - window) if window else 0
        o, l = out[b].double().cpu(), lse[b].double().cpu()
        if n == lo:
            assert (o == 0).all() and (l == float("-inf")).all()
            continue
        k, v = (x[b][lo:n].double().cpu() for x in kv)
        for h in range(q.shape[1]):
            kh, vh, qq = k[:, h // group], v[:, h // group], q[b, h].double().cpu()
            x = scale * (kh @ qq)
            big = abs(scale) * (kh.abs() @ qq.abs())
            p = torch.softmax(x, 0)
            want = p @ vh
            d = float(big.max()) * (2 * split + (qq.numel() + 8) * u) + float(x.abs().max()) * 2 * u
            d += abs(scale) * 2.0 ** -38 * float(qq.abs().max()) * float(kh.abs().sum(-1).max())
            err = 2 * (2 * d + 2.0 ** -20) + (n - lo + 16) * u + 2 * split
            tol = err * (p @ vh.abs()) + half * want.abs() + 1e-30
            if out.dtype == torch.bfloat16 and fmt != "bf16":
                tol += 2.0 ** -11 * (p @ vh.abs())
            if fmt == "f16":
                tol += 2.0 ** -31 * vh.abs().sum(0)
            elif fmt != "bf16":
                tol += (n - lo) * 2.0 ** -29 * (p * vh.abs().amax(-1)).max()
            if out.dtype == torch.float16:
                tol += 2.0 ** -25
            assert ((o[h] - want).abs() <= tol).all(), (b, h, float(((o[h] - want).abs() / tol).max()))
            assert abs(float(l[h]) - float(torch.logsumexp(x, 0))) <= err + 2.0 ** -22 * max(1.0, float(x.abs().max())), (b, h)


def tensors(n, heads, dim, type_, seed):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((n, heads, dim), generator=g) * (1 + 6 * (torch.rand((heads, dim), generator=g) < 0.05))
    v = torch.randn((n, heads, dim), generator=g) * torch.exp2(2 * torch.randn((n, heads, 1), generator=g))
    return k.to(DTYPES[type_]).cuda(), v.to(DTYPES[type_]).cuda()


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
@pytest.mark.parametrize("type_,dim,heads,page", [("f32", 32, 3, 16), ("f16", 64, 1, 48), ("bf16", 96, 2, 32),
                                                  ("f32", 128, 2, 64), ("bf16", 192, 1, 16), ("f16", 256, 2, 128)])
def test_written_values_are_read_back_exactly(fmt, type_, dim, heads, page):
    counts, starts = [1, 0, 37, 16, 130], [0, 5, 3, 16, 31]
    s = Sequences(fmt, dim, heads, page, [a + b for a, b in zip(starts, counts)], seed=dim)
    k, v = tensors(sum(counts), heads, dim, type_, 1)
    s.append(k, v, starts, counts)
    rk, rv = s.read(starts, counts, "f32", fill=-3.0)
    n = sum(counts)
    assert same(rk[:n], stored(k, fmt)) and same(rv[:n], stored(v, fmt))
    assert (rk[n:] == -3).all() and (rv[n:] == -3).all()       # rows behind the last sequence
    for t in ("f16", "bf16"):
        rk, rv = s.read(starts, counts, t)
        assert same(rk, stored(k, fmt).float().to(DTYPES[t])) and same(rv, stored(v, fmt).float().to(DTYPES[t]))
    s.sync()


@pytest.mark.parametrize("fmt", ["f16", "mx8", "mx4"])
def test_token_by_token_equals_one_call(fmt):
    dim, heads, page, n = 64, 2, 16, 35
    k, v = tensors(3 * n, heads, dim, "bf16", 2)
    k, v = k.view(3, n, heads, dim), v.view(3, n, heads, dim)
    s = Sequences(fmt, dim, heads, page, [n] * 3)
    for i in range(n):
        s.append(k[:, i].contiguous(), v[:, i].contiguous(), [i] * 3)      # one token per sequence, no row offsets
    rk, rv = s.read([0] * 3, [n] * 3)
    assert same(rk, stored(k, fmt).view(-1, heads, dim)) and same(rv, stored(v, fmt).view(-1, heads, dim))
    # overwriting in the middle leaves the neighbours alone
    k2, v2 = tensors(3 * 4, heads, dim, "bf16", 3)
    s.append(k2, v2, [14, 0, 31], [4, 4, 4])
    k, v = k.clone(), v.clone()
    for b, st in enumerate([14, 0, 31]):
        k[b, st:st + 4], v[b, st:st + 4] = k2[4 * b:4 * b + 4], v2[4 * b:4 * b + 4]
    rk, rv = s.read([0] * 3, [n] * 3)
    assert same(rk, stored(k, fmt).view(-1, heads, dim)) and same(rv, stored(v, fmt).view(-1, heads, dim))
    s.sync()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_block_scales_at_the_borders(fmt):
    """Zero blocks, values at and next to the largest code times a power of two, ties, subnormals, the largest finite
    values, infinities and NaN (their block only)."""
    top = 448.0 if fmt == "mx8" else 6.0
    rows = []
    for e in (-130, -126, -20, 0, 3, 100, 118):
        base = np.zeros(64, np.float32)
        base[0] = np.float32(top) * np.float32(2.0) ** e if e > -126 else np.float32(2.0 ** e)
        rows.append(base.copy())
        rows.append(np.nextafter(base, np.float32(np.inf), dtype=np.float32) * (base != 0))
        ties = base.copy()
        ties[1:32] = (np.arange(31) - 15) * np.float32(0.125) * np.float32(2.0) ** max(e, -100)
        rows.append(ties)
    rows.append(np.zeros(64, np.float32))
    for bad in (np.inf, -np.inf, np.nan):
        r = np.linspace(-1, 1, 64).astype(np.float32)
        r[40] = bad
        rows.append(r)
    r = np.full(64, np.finfo(np.float32).max, np.float32)
    rows.append(r)
    x = torch.from_numpy(np.stack(rows)).view(-1, 1, 64).cuda()
    n = x.shape[0]
    s = Sequences(fmt, 64, 1, 16, [n])
    s.append(x, -x, [0], [n])
    rk, rv = s.read([0], [n])
    # read back in 32 bits: the largest finite value, (2 - 2^-23) 2^127, is 256 - 2^-15 (mx8) or 4 - 2^-21 (mx4) scales,
    # which rounds up to 2^128 and so reads back as infinity
    want = stored(x, fmt).float()
    assert bool(torch.isinf(want[-1]).all()) and not bool(torch.isinf(want[:-1]).any())
    assert same(rk, want) and same(rv, -want)
    assert torch.isnan(want).sum() == 3 * 32
    s.sync()


CASES = [  # format, type, dim, kv heads, group, page, lengths, window
    ("f16", "f16", 64, 2, 1, 16, [0, 1, 15, 16, 17, 33, 200], 0),
    ("f16", "f32", 128, 2, 4, 32, [129, 0, 64, 1], 0),
    ("f16", "bf16", 128, 1, 3, 48, [100, 47, 48, 49], 0),
    ("f16", "f16", 96, 2, 7, 16, [70, 31], 20),
    ("bf16", "bf16", 64, 3, 8, 16, [40, 0, 129], 0),
    ("bf16", "f32", 256, 1, 2, 64, [77, 300], 0),
    ("bf16", "f16", 32, 2, 9, 16, [33, 90], 16),
    ("mx8", "f16", 128, 2, 4, 16, [1, 0, 16, 77, 513], 0),
    ("mx8", "f32", 64, 1, 16, 32, [100, 31, 32], 0),
    ("mx8", "bf16", 256, 2, 5, 128, [140, 129], 100),
    ("mx8", "f32", 96, 2, 1, 48, [95, 49, 7], 0),
    ("mx8", "f16", 32, 4, 6, 16, [65, 64], 1),
    ("mx4", "bf16", 128, 2, 8, 64, [65, 0, 500, 2], 0),
    ("mx4", "f32", 192, 1, 3, 16, [50, 17], 0),
    ("mx4", "f16", 64, 2, 33, 32, [90, 33], 64),
    ("mx4", "f32", 32, 1, 71, 16, [40], 0),
    ("f16", "f32", 192, 1, 20, 16, [40, 100], 0),
    ("mx8", "f32", 128, 1, 64, 16, [300, 10], 0),
    ("bf16", "bf16", 128, 1, 130, 16, [100, 18], 0),
]


@pytest.mark.parametrize("fmt,type_,dim,heads,group,page,lengths,window", CASES)
def test_attend(fmt, type_, dim, heads, group, page, lengths, window):
    s = Sequences(fmt, dim, heads, page, lengths, seed=7)
    n = sum(lengths)
    k, v = tensors(n, heads, dim, type_, 11)
    s.append(k, v, [0] * len(lengths), lengths)
    q = tensors(len(lengths), heads * group, dim, type_, 12)[0]
    scale = dim ** -0.5
    out, lse = s.attend(q, lengths, scale, window)
    s.sync()
    cut = lambda x: torch.split(stored(x, fmt), lengths)  # noqa: E731
    check_attend(q, (cut(k), cut(v)), lengths, scale, window, fmt, out, lse, group)
    again, lse2 = s.attend(q, lengths, scale, window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)      # same bits every time


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
def test_what_lies_behind_the_length_does_not_count(fmt):
    dim, heads, group, page, cap = 128, 2, 4, 32, 96
    s = Sequences(fmt, dim, heads, page, [cap, cap])
    k, v = tensors(2 * cap, heads, dim, "f32", 4)
    k, v = k.view(2, cap, heads, dim), v.view(2, cap, heads, dim)
    lengths = [41, 64]
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
        k[b, :n - 20], v[b, :n - 20] = float("inf"), float("nan")      # before the window
    s.append(k.view(-1, heads, dim), v.view(-1, heads, dim), [0, 0], [cap, cap])
    q = tensors(2, heads * group, dim, "f32", 5)[0]
    out, lse = s.attend(q, lengths, 0.1, 20)
    check_attend(q, (stored(k, fmt), stored(v, fmt)), lengths, 0.1, 20, fmt, out, lse, group)
    # a value that is not finite reaches the rows of its own head and sequence only
    v2 = v.clone()
    v2[0, 30, 0, 5] = float("nan")
    s.append(k.view(-1, heads, dim), v2.view(-1, heads, dim), [0, 0], [cap, cap])
    out2, _ = s.attend(q, lengths, 0.1, 20)
    assert torch.isnan(out2[0, :group, 5]).all()
    assert torch.equal(out2[0, group:], out[0, group:]) and torch.equal(out2[1], out[1])
    if fmt.startswith("mx"):   # the block of the value, nothing else
        assert torch.isnan(out2[0, :group, :32]).all() and torch.equal(out2[0, :group, 32:], out[0, :group, 32:])
    s.sync()


@pytest.mark.parametrize("fmt", ["f16", "mx8", "mx4"])
def test_magnitudes_far_apart(fmt):
    """Large and small queries, keys and values; scores far apart; value scales that grow along the sequence."""
    dim, heads, n = 64, 1, 150
    s = Sequences(fmt, dim, heads, 16, [n])
    g = torch.Generator().manual_seed(9)
    k = torch.randn((n, heads, dim), generator=g).cuda()
    grow = torch.linspace(-12, 12, n).view(n, 1, 1).cuda()
    v = torch.randn((n, heads, dim), generator=g).cuda() * torch.exp2(grow)
    s.append(k, v, [0], [n])
    for big in (1e-30, 1e-3, 1.0, 1e4):
        q = (torch.randn((1, 3, dim), generator=g) * big).cuda()
        scale = 0.5 / big if big != 1.0 else 2.0
        out, lse = s.attend(q, [n], scale)
        check_attend(q, ([stored(k, fmt)], [stored(v, fmt)]), [n], scale, 0, fmt, out, lse, 3)
    if fmt != "f16":   # the scale's whole range
        s.append(k * 2.0 ** 90, v * 2.0 ** -100, [0], [n])
        q = (torch.randn((1, 3, dim), generator=g) * 2.0 ** -90).cuda()
        out, lse = s.attend(q, [n], 1.0)
        check_attend(q, ([stored(k * 2.0 ** 90, fmt)], [stored(v * 2.0 ** -100, fmt)]), [n], 1.0, 0, fmt, out, lse, 3)
    s.sync()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("dim", [64, 96, 192, 256])
def test_blocks_of_one_token_far_apart(fmt, dim):
    """Value blocks 2^13 to 2^20 below the token's largest, blocks of zeros, and a token whose values are all zero: the
    small blocks come out with the accuracy of their own size as long as the floor of the split allows."""
    n, blocks = 70, dim // 32
    s = Sequences(fmt, dim, 1, 16, [n])
    g = torch.Generator().manual_seed(dim)
    k = torch.randn((n, 1, dim), generator=g).cuda()
    low = torch.randint(0, 21, (n, 1, blocks), generator=g).float()
    low[:, :, 0] = 0
    low[: n // 2] = low[: n // 2].clamp(max=13)           # a stretch of ordinary tokens first
    v = torch.randn((n, 1, blocks, 32), generator=g) * torch.exp2(-low)[..., None]
    v[5, :, blocks - 1] = 0
    v[40, :, 0] = 0
    v[41] = 0
    v = v.reshape(n, 1, dim).cuda()
    s.append(k, v, [0], [n])
    rk, rv = s.read([0], [n])
    assert same(rv, stored(v, fmt)) and same(rk, stored(k, fmt))
    q = torch.randn((1, 2, dim), generator=g).cuda()
    out, lse = s.attend(q, [n], dim ** -0.5)
    check_attend(q, ([stored(k, fmt)], [stored(v, fmt)]), [n], dim ** -0.5, 0, fmt, out, lse, 2)
    s.sync()


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
@pytest.mark.parametrize("size", [1e9, 1e12, 1e30])
def test_scores_past_the_integers_of_fp32(fmt, size):
    """Scores of 1e9 and more are further apart than their weights' range, or the same: two tokens, in different parts of
    the work, share all of the weight, and the others have none.  Equal keys give equal scores and weights, so what is
    left is the split of the weights (2^-22, bf16 2^-16, in numerator and denominator) and a few roundings of fp32.  The
    score itself carries the query's split (1e9 is not a sum of two 8-bit numbers: 2^-17 for bf16) and fp32's roundings."""
    dim, n = 64, 300
    _, v = tensors(n, 1, dim, "f16", 5)
    v = stored(v, fmt).half()
    for sign in (1.0, -1.0):
        k = torch.zeros((n, 1, dim), device="cuda", dtype=torch.float16)
        k[:, 0, 0] = 3.0
        k[[5, 290], 0, 0] = 6.0 if sign > 0 else 1.5   # (exact in every format)
        s = Sequences(fmt, dim, 1, 16, [n])
        s.append(k, v, [0], [n])
        q = torch.zeros((1, 2, dim), device="cuda")
        q[0, :, 0] = torch.tensor([sign * size, 0.0])
        out, lse = s.attend(q, [n], 1.0)
        s.sync()
        two = v[[5, 290], 0].double()
        tol = (2.0 ** -14 if fmt == "bf16" else 2.0 ** -20) * two.abs().mean(0) + 2.0 ** -24 * two.abs().amax()
        assert ((out[0, 0].double() - two.mean(0)).abs() <= tol).all()
        top = (6.0 if sign > 0 else -1.5) * size
        assert abs(float(lse[0, 0]) - (top + np.log(2.0))) <= (2.0 ** -16 if fmt == "bf16" else 2.0 ** -21) * abs(top)
        check_attend(q[:, 1:], [k[None], v[None]], [n], 1.0, 0, fmt, out[:, 1:], lse[:, 1:], 1)


def test_strided_and_unaligned_tensors():
    """Views into one fused projection [tokens, (Hq + 2 Hk) dim], and tensors that start at an odd element."""
    dim, heads, group, n = 64, 2, 3, 50
    width = (heads * group + 2 * heads) * dim
    for shift, type_ in ((0, "f16"), (1, "f16"), (1, "f32"), (3, "bf16")):
        buf = torch.randn(n * width + shift, generator=torch.Generator().manual_seed(3)).to(DTYPES[type_]).cuda()
        es = buf.element_size()
        fused = buf[shift:].view(n, width)
        qo, ko, vo = 0, heads * group * dim, (heads * group + heads) * dim
        s = Sequences("mx8", dim, heads, 16, [n])
        cu, st = s._ints([0, n]), s._ints([0])
        base = buf.data_ptr() + shift * es
        s.cache.append_device(base + ko * es, base + vo * es, type_, n, 1, s.table.data_ptr(), s.max_pages, st.data_ptr(),
                              cu.data_ptr(), (width, dim, width, dim), torch.cuda.current_stream().cuda_stream)
        k = fused[:, ko:vo].reshape(n, heads, dim)
        v = fused[:, vo:].reshape(n, heads, dim)
        rk, rv = s.read([0], [n])
        assert same(rk, stored(k, "mx8")) and same(rv, stored(v, "mx8"))
        q = fused[n - 1:, qo:ko]
        out, lse = s.attend(q, [n], 0.125, query_strides=(width, dim), shape=(1, heads * group, dim))
        check_attend(q.reshape(1, heads * group, dim), ([stored(k, "mx8")], [stored(v, "mx8")]), [n], 0.125, 0, "mx8", out, lse, group)
        s.sync()


def test_odd_strides_both_ways():
    """Rows at odd distances, written from and read back into larger buffers; what lies between the rows stays."""
    dim, heads, n = 96, 2, 37
    for type_ in ("f16", "f32"):
        token, head = heads * (dim + 3) + 5, dim + 3
        buf = torch.randn(n * token + 8, generator=torch.Generator().manual_seed(4)).to(DTYPES[type_]).cuda()
        view = torch.as_strided(buf, (n, heads, dim), (token, head, 1), 1)
        s = Sequences("mx8", dim, heads, 16, [n + 3])
        cu, st = s._ints([0, n]), s._ints([3])
        at = buf.data_ptr() + buf.element_size()
        stream = torch.cuda.current_stream().cuda_stream
        s.cache.append_device(at, at, type_, n, 1, s.table.data_ptr(), s.max_pages, st.data_ptr(), cu.data_ptr(), (token, head) * 2, stream)
        out = torch.full_like(buf, 5.0)
        val = torch.full_like(buf, 6.0)
        es = buf.element_size()
        s.cache.read_device(out.data_ptr() + es, val.data_ptr() + es, type_, n, 1, s.table.data_ptr(), s.max_pages, st.data_ptr(),
                            cu.data_ptr(), (token, head) * 2, stream)
        torch.cuda.synchronize()
        want = stored(view, "mx8").float().to(DTYPES[type_])
        for got, fill in ((out, 5.0), (val, 6.0)):
            assert same(torch.as_strided(got, (n, heads, dim), (token, head, 1), 1), want)
            torch.as_strided(got, (n, heads, dim), (token, head, 1), 1).fill_(fill)
            assert (got == fill).all()
        s.sync()


def test_scales_of_any_sign_no_lse_and_rows_that_are_not_finite():
    dim, heads, group, lengths = 64, 2, 12, [50, 17, 200]
    for fmt in ("f16", "mx4"):
        s = Sequences(fmt, dim, heads, 16, lengths)
        k, v = tensors(sum(lengths), heads, dim, "f32", 8)
        s.append(k, v, [0] * 3, lengths)
        cut = lambda x: torch.split(stored(x, fmt), lengths)  # noqa: E731
        q = tensors(3, heads * group, dim, "f32", 9)[0]
        for scale in (0.0, -0.2, 0.5):
            out, lse = s.attend(q, lengths, scale)
            check_attend(q, (cut(k), cut(v)), lengths, scale, 0, fmt, out, lse, group)
        n = s._ints(lengths)
        again = torch.empty_like(out)
        s.cache.attend_device(q.data_ptr(), "f32", heads * group, 3, s.table.data_ptr(), s.max_pages, n.data_ptr(),
                              again.data_ptr(), 0.5, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(again, out)
        # a query that is not finite spoils its own row only
        bad = q.clone()
        bad[1, 3, 7] = float("nan")
        bad[2, 15, 0] = float("inf")
        got, _ = s.attend(bad, lengths, 0.5)
        hit = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
        hit[1, 3] = hit[2, 15] = True
        assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], out[~hit])
        s.sync()


def test_many_sequences_and_units():
    """More sequences than threads of a CTA, most of them empty or one token long."""
    dim, heads, batch = 32, 2, 1500
    rng = np.random.default_rng(3)
    lengths = [int(x) for x in rng.choice([0, 0, 1, 2, 16, 17, 40], size=batch)]
    s = Sequences("mx8", dim, heads, 16, lengths)
    k, v = tensors(sum(lengths), heads, dim, "f16", 13)
    s.append(k, v, [0] * batch, lengths)
    q = tensors(batch, heads * 2, dim, "f16", 14)[0]
    out, lse = s.attend(q, lengths, 0.25)
    s.sync()
    cut = lambda x: torch.split(stored(x, "mx8"), lengths)  # noqa: E731
    check_attend(q, (cut(k), cut(v)), lengths, 0.25, 0, "mx8", out, lse, 2)


@pytest.mark.parametrize("batch,heads,lengths", [(1, 8, [300]), (37, 8, [200, 0, 193, 208]), (296, 1, [17, 1, 0, 32]),
                                                 (10, 8, [700, 1, 40]), (96, 1, [1000, 64])])
def test_units_left_whole_and_cut(batch, heads, lengths):
    """Batches on both sides of the choice of where the work is cut, with windows that cut them shorter again."""
    dim, group = 64, 3
    lengths = [lengths[i % len(lengths)] for i in range(batch)]
    s = Sequences("f16", dim, heads, 32, lengths)
    k, v = tensors(sum(lengths), heads, dim, "f16", 17)
    s.append(k, v, [0] * batch, lengths)
    q = tensors(batch, heads * group, dim, "f16", 18)[0]
    cut = lambda x: torch.split(stored(x, "f16"), lengths)  # noqa: E731
    kv = cut(k), cut(v)
    for window in (0, 90):
        out, lse = s.attend(q, lengths, 0.1, window)
        s.sync()
        check_attend(q, kv, lengths, 0.1, window, "f16", out, lse, group)
        again, lse2 = s.attend(q, lengths, 0.1, window)
        assert same(out, again) and same(lse, lse2)


@pytest.mark.parametrize("fmt,type_,dim,heads,group", [("f16", "f16", 128, 1, 4), ("bf16", "bf16", 256, 1, 16), ("mx8", "f32", 128, 2, 1),
                                                       ("mx4", "bf16", 64, 1, 33)])
def test_one_long_sequence_over_all_ctas(fmt, type_, dim, heads, group):
    """Units that every CTA holds a part of: joined by neighbours first, then over the groups."""
    n = 40000 + 13
    s = Sequences(fmt, dim, heads, 64, [n, 5], seed=2)
    k, v = tensors(n + 5, heads, dim, type_, 15)
    s.append(k, v, [0, 0], [n, 5])
    q = tensors(2, heads * group, dim, type_, 16)[0]
    scale = 3 * dim ** -0.5
    out, lse = s.attend(q, [n, 5], scale)
    s.sync()
    cut = lambda x: torch.split(stored(x, fmt), [n, 5])  # noqa: E731
    check_attend(q, (cut(k), cut(v)), [n, 5], scale, 0, fmt, out, lse, group)
    again, lse2 = s.attend(q, [n, 5], scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_bad_pages_and_lengths_are_reported_and_left_out():
    import eos_b200
    dim, heads, n = 64, 2, 64
    s = Sequences("f16", dim, heads, 16, [n, n])
    k, v = tensors(2 * n, heads, dim, "f16", 6)
    s.append(k, v, [0, 0], [n, n])
    s.sync()
    q = tensors(2, heads, dim, "f16", 7)[0]
    good, _ = s.attend(q, [n, n], 0.1)
    table = s.table.clone()
    for page in (-1, s.pages, 2 ** 31 - 1):
        s.table.copy_(table)
        s.table[0, 1] = page
        out, lse = s.attend(q, [n, n], 0.1)
        with pytest.raises(eos_b200.EosB200DeviceStatusError, match="page"):
            s.sync()
        s.sync()                                         # reported once
        assert torch.equal(out[1], good[1])
        keep = torch.cat([torch.arange(16), torch.arange(32, n)])
        check_attend(q[:1], ([k[:n][keep]], [v[:n][keep]]), [n - 16], 0.1, 0, "f16", out[:1], lse[:1], 1)
        # an append skips that page and writes the others
        s.append(torch.zeros_like(k), v, [0, 0], [n, n])
        with pytest.raises(eos_b200.EosB200DeviceStatusError):
            s.sync()
        rk, _ = s.read([0, 0], [n, n], "f16", fill=9.0)
        with pytest.raises(eos_b200.EosB200DeviceStatusError):
            s.sync()
        assert (rk[16:32] == 9).all() and (rk[:16] == 0).all() and (rk[32:2 * n] == 0).all()
        s.table.copy_(table)
        assert torch.equal(s.read([0, 0], [n, n], "f16")[0][16:32], k[16:32])
        s.append(k, v, [0, 0], [n, n])
        s.sync()
    for lengths in ([-5, n], [s.max_pages * 16 + 1, n]):
        out, _ = s.attend(q, lengths, 0.1)
        with pytest.raises(eos_b200.EosB200DeviceStatusError):
            s.sync()
        assert torch.equal(out[1], good[1])
        if lengths[0] < 0:
            assert (out[0] == 0).all()
    # row offsets that run backwards or past the rows, starts behind the table
    for counts, starts in (([-3, 5], [0, 0]), ([2 * n, n], [0, 0]), ([4, 4], [-1, 0]), ([4, 4], [2 ** 31 - 3, 0]), ([4, 4], [s.max_pages * 16 - 2, 0])):
        s.append(k, v, starts, counts)
        with pytest.raises(eos_b200.EosB200DeviceStatusError):
            s.sync()
        s.append(k, v, [0, 0], [n, n])
        s.sync()
        assert torch.equal(s.read([0, 0], [n, n], "f16")[0], k)


def test_refusals():
    import eos_b200
    rt = eos_b200.Runtime(0)
    E = eos_b200.EosB200Error
    for args, what in (((1, 8, 1, 64, "f16"), "page_size"), ((1, 24, 1, 64, "f16"), "page_size"), ((1, 16, 0, 64, "f16"), "kv_heads"),
                       ((0, 16, 1, 64, "f16"), "pages"), ((1, 16, 1, 80, "f16"), "head_dim"), ((1, 16, 1, 512, "mx8"), "head_dim"),
                       ((2 ** 31 - 1, 65536, 64, 256, "f16"), "memory")):
        with pytest.raises(E, match=what):
            eos_b200.KvCache(rt, *args)
    c = eos_b200.KvCache(rt, 4, 16, 2, 64, "mx8")
    assert c.page_bytes == 2 * 16 * 2 * (64 + 2) + 2 * 32      # codes and scales, and 32 bytes a record of 16 tokens
    x = torch.zeros((4, 2, 64), device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    p, t = x.data_ptr(), i.data_ptr()
    with pytest.raises(ValueError, match="element type"):
        c.append_device(p, p, "f64", 1, 1, t, 1, t)
    for call in (lambda **k: c.append_device(**k), lambda **k: c.read_device(**k)):
        ok = dict(d_key=p, d_value=p, type="f32", tokens=1, batch=1, d_page_table=t, max_pages=1, d_starts=t)
        for bad in (dict(type=3), dict(tokens=-1), dict(batch=-1), dict(tokens=2), dict(d_key=None), dict(d_value=None),
                    dict(d_page_table=None), dict(d_starts=None), dict(max_pages=0), dict(strides=(-1, 64, 128, 64)),
                    dict(d_key=p + 1), dict(tokens=2 ** 31, d_cu_tokens=t)):
            with pytest.raises(E):
                call(**{**ok, **bad})
        assert call(**{**ok, "tokens": 0, "batch": 0}) == 0
        assert call(**{**ok, "tokens": 0, "d_cu_tokens": t}) == 0
    ok = dict(d_query=p, type="f32", q_heads=2, batch=1, d_page_table=t, max_pages=1, d_lengths=t, d_out=p, scale=1.0)
    for bad in (dict(type=-1), dict(q_heads=3), dict(q_heads=0), dict(batch=-1), dict(d_query=None), dict(d_page_table=None),
                dict(d_lengths=None), dict(d_out=None), dict(max_pages=0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(window=-1), dict(query_strides=(-1, 64)), dict(d_out=p + 2)):
        with pytest.raises(E):
            c.attend_device(**{**ok, **bad})
    assert c.attend_device(**{**ok, "batch": 0}) == 0
    c.close()
    c.close()
    rt.close()


def test_a_decoding_loop_on_a_stream_and_in_a_graph():
    """Prompt, then tokens one by one: append, attend, lengths advanced on the device -- eagerly on a side stream, and as
    one captured step that is replayed, in turn with eager calls of another cache of the same runtime."""
    import eos_b200
    dim, heads, group, page, prompt, steps = 128, 2, 4, 32, [45, 0, 130], 40
    batch = len(prompt)
    rt = eos_b200.Runtime(0)
    k, v = tensors(sum(prompt), heads, dim, "bf16", 21)
    sk, sv = tensors(steps * batch, heads, dim, "bf16", 22)
    sq = tensors(steps * batch, heads * group, dim, "bf16", 23)[0]
    sk, sv, sq = sk.view(steps, batch, heads, dim), sv.view(steps, batch, heads, dim), sq.view(steps, batch, heads * group, dim)
    results = []
    stream = torch.cuda.Stream()
    for graph in (False, True):
        s = Sequences("mx8", dim, heads, page, [n + steps for n in prompt], runtime=rt)
        other = Sequences("mx4", dim, heads, page, [64] * batch, runtime=rt)
        s.append(k, v, [0] * batch, prompt)
        at, n = s._ints(prompt), s._ints(prompt) + 1
        ik, iv, iq = sk[0].clone(), sv[0].clone(), sq[0].clone()
        out = torch.empty((batch, heads * group, dim), dtype=torch.bfloat16, device="cuda")
        lse = torch.empty((batch, heads * group), device="cuda")
        outs, lses = [], []

        def step(handle):
            s.cache.append_device(ik.data_ptr(), iv.data_ptr(), "bf16", batch, batch, s.table.data_ptr(), s.max_pages,
                                  at.data_ptr(), stream=handle)
            s.cache.attend_device(iq.data_ptr(), "bf16", heads * group, batch, s.table.data_ptr(), s.max_pages, n.data_ptr(),
                                  out.data_ptr(), dim ** -0.5, d_lse=lse.data_ptr(), stream=handle)
            at.add_(1)
            n.add_(1)

        torch.cuda.synchronize()
        captured = None
        if graph:
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=stream):
                step(stream.cuda_stream)
        with torch.cuda.stream(stream):
            for i in range(steps):
                ik.copy_(sk[i]), iv.copy_(sv[i]), iq.copy_(sq[i])
                if captured is not None:
                    captured.replay()
                else:
                    step(stream.cuda_stream)
                outs.append(out.clone()), lses.append(lse.clone())
                if i % 7 == 0:
                    zero = torch.zeros(batch, dtype=torch.int32, device="cuda")
                    other.cache.append_device(ik.data_ptr(), iv.data_ptr(), "bf16", batch, batch, other.table.data_ptr(),
                                              other.max_pages, zero.data_ptr(), stream=stream.cuda_stream)
        stream.synchronize()
        s.cache.sync(stream.cuda_stream)
        results.append((torch.stack(outs), torch.stack(lses)))
        del captured
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    kk, vv = torch.split(k, prompt), torch.split(v, prompt)
    for i in (0, 1, 17, steps - 1):
        fk = [stored(torch.cat([kk[b], sk[:i + 1, b]]), "mx8") for b in range(batch)]
        fv = [stored(torch.cat([vv[b], sv[:i + 1, b]]), "mx8") for b in range(batch)]
        check_attend(sq[i], (fk, fv), [p + i + 1 for p in prompt], dim ** -0.5, 0, "mx8", results[0][0][i], results[0][1][i], group)


def test_shared_pages():
    """Two sequences with a common prefix share its pages."""
    dim, heads, page = 64, 1, 16
    s = Sequences("mx4", dim, heads, page, [64, 64])
    k, v = tensors(64, heads, dim, "f16", 31)
    s.table[1, :2] = s.table[0, :2]
    s.append(torch.cat([k, k[32:] * 2]), torch.cat([v, v[32:]]), [0, 32], [64, 32])
    q = tensors(1, 2, dim, "f16", 32)[0].repeat(2, 1, 1)
    out, lse = s.attend(q, [64, 60], 0.2)
    second = stored(torch.cat([k[:32], k[32:] * 2]), "mx4")
    check_attend(q, ([stored(k, "mx4"), second], [stored(v, "mx4")] * 2), [64, 60], 0.2, 0, "mx4", out, lse, 2)
    s.sync()


@pytest.mark.parametrize("fmt", ["f16", "mx4"])
def test_offsets_past_32_bits(fmt):
    """A cache of 5 GiB whose last pages are used, and rows and queries 2^28 and 2^30 elements apart."""
    import eos_b200
    dim, heads, page, n = 128, 2, 64, 17
    rt = eos_b200.Runtime(0)
    probe = eos_b200.KvCache(rt, 1, page, heads, dim, fmt)
    pages = (5 << 30) // probe.page_bytes
    probe.close()
    cache = eos_b200.KvCache(rt, pages, page, heads, dim, fmt)
    far = torch.zeros((1 << 32) + (1 << 16), dtype=torch.float16, device="cuda")
    step = 1 << 28
    key = torch.as_strided(far, (n, heads, dim), (step - 8, dim, 1), 0)
    value = torch.as_strided(far, (n, heads, dim), (step - 8, dim, 1), heads * dim)
    k, v = tensors(n, heads, dim, "f16", 31)
    key.copy_(k)
    value.copy_(v)
    table = torch.tensor([[pages - 1], [pages - 3], [1], [pages - 2]], dtype=torch.int32, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, starts, lengths = ints(0, 5, 5, 11, 17), ints(0, 0, 0, 0), ints(5, 0, 6, 6)
    st = torch.cuda.current_stream().cuda_stream
    strides = (step - 8, dim, step - 8, dim)
    cache.append_device(key.data_ptr(), value.data_ptr(), "f16", n, 4, table.data_ptr(), 1, starts.data_ptr(), cu.data_ptr(),
                        strides, st)
    far.zero_()
    cache.read_device(key.data_ptr(), value.data_ptr(), "f16", n, 4, table.data_ptr(), 1, starts.data_ptr(), cu.data_ptr(),
                      strides, st)
    sk, sv = stored(k, fmt), stored(v, fmt)
    assert same(key, sk.half()) and same(value, sv.half())
    far.zero_()
    q0 = tensors(4, heads * 3, dim, "f16", 32)[0]
    q = torch.as_strided(far, q0.shape, ((1 << 30) + 8, dim, 1), 0)
    q.copy_(q0)
    out, lse = torch.empty_like(q0), torch.empty(q0.shape[:2], device="cuda")
    cache.attend_device(q.data_ptr(), "f16", heads * 3, 4, table.data_ptr(), 1, lengths.data_ptr(), out.data_ptr(), 0.1, 0,
                        lse.data_ptr(), ((1 << 30) + 8, dim), st)
    cache.sync(st)
    cut = lambda x: torch.split(x, [5, 0, 6, 6])  # noqa: E731
    check_attend(q0, (cut(sk), cut(sv)), [5, 0, 6, 6], 0.1, 0, fmt, out, lse, 3)
    cache.close()


def test_two_caches_at_once():
    """Attends, appends and reads of two caches, eager and replayed, on two streams that nothing orders."""
    import eos_b200
    rt = eos_b200.Runtime(0)
    dim, heads, lengths = 64, 2, [5000, 700, 33]
    made = []
    for i in range(2):
        s = Sequences("mx8", dim, heads, 32, [x + 1 for x in lengths], seed=i, runtime=rt)
        k, v = tensors(sum(lengths), heads, dim, "f16", 40 + i)
        s.append(k, v, [0, 0, 0], lengths)
        q = tensors(3, heads * 4, dim, "bf16", 50 + i)[0]
        want, lse = s.attend(q, lengths, 0.125)
        made.append((s, k, v, q, want, lse, torch.cuda.Stream(), s._ints(lengths), s._ints([0, 0, 0]), s._ints(np.cumsum([0] + lengths))))
    results = []
    graphs = []

    def step(m, out, lse, rk, rv):
        s, k, v, q, _, _, stream, n, zero, cu = m
        at = torch.cuda.current_stream().cuda_stream
        s.cache.append_device(k.data_ptr(), v.data_ptr(), "f16", k.shape[0], 3, s.table.data_ptr(), s.max_pages, zero.data_ptr(),
                              cu.data_ptr(), stream=at)
        s.cache.attend_device(q.data_ptr(), "bf16", heads * 4, 3, s.table.data_ptr(), s.max_pages, n.data_ptr(), out.data_ptr(),
                              0.125, 0, lse.data_ptr(), stream=at)
        s.cache.read_device(rk.data_ptr(), rv.data_ptr(), "f16", k.shape[0], 3, s.table.data_ptr(), s.max_pages, zero.data_ptr(),
                            cu.data_ptr(), stream=at)

    for m in made:
        outs = [(torch.zeros_like(m[4]), torch.zeros_like(m[5]), torch.zeros_like(m[1]), torch.zeros_like(m[2])) for _ in range(2)]
        results.append(outs)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=m[6]):
            step(m, *outs[1])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for m, outs, g in zip(made, results, graphs):
            with torch.cuda.stream(m[6]):
                step(m, *outs[0])
                g.replay()
    torch.cuda.synchronize()
    for m, outs in zip(made, results):
        for out, lse, rk, rv in outs:
            assert same(out, m[4]) and same(lse, m[5])
            assert same(rk, stored(m[1], "mx8").half()) and same(rv, stored(m[2], "mx8").half())
        m[0].sync()
