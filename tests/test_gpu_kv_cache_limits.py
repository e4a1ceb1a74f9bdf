"""Paged key-value cache on the device, at the limits of what its calls allow: the bits that results carry, the range of
scores and lengths, errors and workspaces of caches that live side by side."""
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_kv_cache import DTYPES, Sequences, check_attend, same, stored, tensors  # noqa: E402


def formula(q, k, v, scale, group):
    """out, lse in 64 bits of one sequence, p @ |v| and the largest |score| of every row: q [heads * group, dim];
    k, v [n, heads, dim]."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    rows = []
    for h in range(q.shape[0]):
        kh, vh = k[:, h // group], v[:, h // group]
        x = scale * (kh @ q[h])
        p = torch.softmax(x, 0)
        rows.append((p @ vh, torch.logsumexp(x, 0), p @ vh.abs(), x.abs().max()))
    return [torch.stack([r[i] for r in rows]) for i in range(4)]


def whole(shape, type_, seed):
    """Whole numbers from -2 to 2, exact in every type and format: their products' sums are exact too."""
    return torch.randint(-2, 3, shape, generator=torch.Generator().manual_seed(seed)).to(DTYPES[type_]).cuda()


@pytest.mark.parametrize("fmt,dim,group,n", [("f16", 64, 2, 16), ("f16", 128, 9, 5), ("mx8", 128, 4, 16), ("mx8", 96, 12, 33),
                                             ("mx4", 128, 8, 16), ("mx4", 256, 3, 5)])
def test_bf16_results_are_the_rounding_of_a_result_in_32_bits(fmt, dim, group, n):
    """The weights of bf16 results carry the 22 bits that all others do.  The dot products here are exact, so a score is off
    by the roundings of its scale, of its product with it and of its distance from the maximum, 2^-22 |x| with room, a
    weight by twice that and 2^-20 (exp2), n additions by u = 2^-23 each and the weights' split by 2^-22, in numerator and
    denominator.  The split's floor, 2^-25 below f16's normal numbers, is 2^-31 sum |v| (f16) or n 2^-29 max|v|
    (block scales).  What is left is the one rounding to bf16."""
    heads, scale, u = 2, 2.0 ** -4, 2.0 ** -23
    s = Sequences(fmt, dim, heads, 32, [n])
    k, v = whole((n, heads, dim), "bf16", 61), tensors(n, heads, dim, "bf16", 62)[1]
    s.append(k, v, [0], [n])
    q = whole((1, heads * group, dim), "bf16", 63)
    out, _ = s.attend(q, [n], scale)
    s.sync()
    sv = stored(v, fmt)
    want, _, size, top = formula(q[0], k, sv, scale, group)
    tol = (2 * (2 * 2.0 ** -22 * top + 2.0 ** -20) + (n + 16) * u + 2 * 2.0 ** -22)[:, None] * size
    tol += 2.0 ** -31 * n * sv.abs().max().item() * (1 if fmt == "f16" else 4)
    got = out[0].double().cpu()
    low, high = ((want - tol).float().bfloat16().double(), (want + tol).float().bfloat16().double())
    assert ((got >= low) & (got <= high)).all(), float(((got < low) | (got > high)).double().mean())


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
@pytest.mark.parametrize("dim,group", [(64, 5), (128, 16), (256, 3)])
def test_queries_in_32_bits_keep_them(fmt, dim, group):
    """Keys with one element that is not zero: a score is one product, of a number of 24 bits and 1.  It is off by the
    query's split (f16: 11 + 11 bits, 2^-22 with room; bf16: three times 8, less), the sum of the parts (2 u, u = 2^-23) and the roundings of the scale,
    its product and the distance to the maximum: 2^-22 + 4 u = 2^-20.7 of |x|, here below 2^-20.  lse carries it once and
    exp2's 2^-22, out twice (weight and sum), with 2^-22 from the weights' split, the sums' 32 u and the split's floor, n 2^-29 max|v|."""
    heads, n, scale, u = 1, 16, 8.0, 2.0 ** -23
    s = Sequences(fmt, dim, heads, 16, [n])
    k = torch.zeros((n, heads, dim), device="cuda")
    k[torch.arange(n), 0, torch.arange(n) * (dim // n) + 1] = 1.0
    v = tensors(n, heads, dim, "f32", 71)[1]
    s.append(k, v, [0], [n])
    q = torch.randn((1, heads * group, dim), generator=torch.Generator().manual_seed(72)).cuda()
    out, lse = s.attend(q, [n], scale)
    s.sync()
    sv = stored(v, fmt)
    want, wanted, size, top = formula(q[0], k, sv, scale, group)
    d = 2.0 ** -20 * top
    assert ((lse[0].double().cpu() - wanted).abs() <= d + 2.0 ** -21 + 2.0 ** -22 * wanted.abs()).all()
    tol = (4 * d + 4 * 2.0 ** -22 + 32 * u)[:, None] * size + n * 2.0 ** -29 * sv.abs().max().item()
    assert ((out[0].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
def test_a_single_token_gives_its_value(fmt):
    """Whatever its score, the weight is divided by itself: what is left is its split (f16 2^-24, bf16 in three parts less),
    the sum of the parts (3 u, u = 2^-23), the approximate quotient (2 u), two products (u), and for block scales one more
    rounding of exp2's argument (ln 2 2^-21, 3 u)."""
    dim, rows = 64, 64
    s = Sequences(fmt, dim, 1, 16, [1])
    k, v = tensors(1, 1, dim, "f32", 73)
    s.append(k, v, [0], [1])
    q = torch.randn((1, rows, dim), generator=torch.Generator().manual_seed(74)).cuda()
    out, _ = s.attend(q, [1], 0.3)
    s.sync()
    sv = stored(v, fmt)[0, 0]
    assert ((out[0].double() - sv).abs() <= 12 * 2.0 ** -23 * sv.abs()).all()


def test_errors_stay_with_their_cache():
    """What a call on one cache met is reported by that cache's sync, once, whatever else its runtime runs meanwhile, and by no other's."""
    import eos_b200
    from eos_b200 import synth
    dim, heads, n = 64, 2, 40
    rt = eos_b200.Runtime(0)
    a, b = (Sequences(fmt, dim, heads, 16, [n], seed=i, runtime=rt) for i, fmt in enumerate(("f16", "mx8")))
    k, v = tensors(n, heads, dim, "f16", 81)
    q = tensors(1, heads, dim, "f16", 82)[0]
    encoder = eos_b200.BertEmbedder(rt, **synth.make_q8_encoder(1, 128, 2, 256, vocab=200, max_pos=64, seed=1, head_out=64))
    ids, mask, _ = synth.make_batch(2, 16, 200, 5, 16, seed=2)
    error = eos_b200.EosB200DeviceStatusError

    def others():
        b.append(k, v, [0], [n])
        b.attend(q, [n], 0.1)
        b.read([0], [n], "f16")
        b.sync()
        encoder.run(ids, mask)

    good = a.table.clone()
    a.append(k, v, [0], [n])
    a.sync()
    for call, what in ((lambda: a.append(k, v, [0], [n]), "page"), (lambda: a.read([0], [n], "f16"), "page"),
                       (lambda: a.attend(q, [n], 0.1), "page"), (lambda: a.append(k, v, [-1], [n]), "start")):
        a.table.copy_(good)
        if what == "page":
            a.table[0, 1] = a.pages
        call()
        others()
        with pytest.raises(error, match=what):
            a.sync()
        a.sync()
        others()
    # both at once
    a.table[0, 0] = -1
    a.attend(q, [n], 0.1)
    b.attend(q, [-1], 0.1)
    with pytest.raises(error, match="length"):
        b.sync()
    with pytest.raises(error, match="page"):
        a.sync()
    # two kinds in one cache are both named
    a.attend(q, [n], 0.1)
    a.attend(q, [-7], 0.1)
    with pytest.raises(error, match="page.*length"):
        a.sync()
    a.sync()
    b.sync()
    encoder.close()


def test_the_longest_sequences():
    """Positions up to 2^31 - 2 and a length of 2^31 - 1, the largest there are, on pages that a table names again and again;
    another sequence of the call is not touched by it."""
    import eos_b200
    rt = eos_b200.Runtime(0)
    dim, heads, group, page, wide, last, n = 32, 1, 3, 65536, 32768, 2 ** 31 - 1, 1000
    cache = eos_b200.KvCache(rt, 3, page, heads, dim, "mx8")
    table = torch.zeros((2, wide), dtype=torch.int32, device="cuda")
    table[0, -1], table[1] = 1, 2
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = tensors(n + 40, heads, dim, "f32", 91)
    q = tensors(2, group, dim, "f32", 92)[0]
    st = torch.cuda.current_stream().cuda_stream
    starts, cu, lengths = ints(last - n, 0), ints(0, n, n + 40), ints(last, 40)
    cache.append_device(k.data_ptr(), v.data_ptr(), "f32", n + 40, 2, table.data_ptr(), wide, starts.data_ptr(), cu.data_ptr(), stream=st)
    rk, rv = torch.zeros_like(k), torch.zeros_like(v)
    cache.read_device(rk.data_ptr(), rv.data_ptr(), "f32", n + 40, 2, table.data_ptr(), wide, starts.data_ptr(), cu.data_ptr(), stream=st)
    cache.sync(st)
    sk, sv = stored(k, "mx8"), stored(v, "mx8")
    assert same(rk, sk) and same(rv, sv)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    for window in (1, 333, n):
        cache.attend_device(q.data_ptr(), "f32", group, 2, table.data_ptr(), wide, lengths.data_ptr(), out.data_ptr(), 0.2, window,
                            lse.data_ptr(), stream=st)
        cache.sync(st)
        spans = [(sk[n - window:n], sk[n:][-min(window, 40):]), (sv[n - window:n], sv[n:][-min(window, 40):])]
        check_attend(q, spans, [min(window, n), min(window, 40)], 0.2, 0, "mx8", out, lse, group)
    # all of it: 2^31 - 1 - n tokens of zeros, whose weights are 1, and the last n
    cache.attend_device(q.data_ptr(), "f32", group, 2, table.data_ptr(), wide, lengths.data_ptr(), out.data_ptr(), 0.2, 0, lse.data_ptr(),
                        stream=st)
    cache.sync(st)
    check_attend(q[1:], [sk[n:][None], sv[n:][None]], [40], 0.2, 0, "mx8", out[1:], lse[1:], group)
    p = torch.exp(0.2 * (sk[:n, 0] @ q[0].double().T))           # [n, group]
    total = last - n + p.sum(0)
    # weights and sums as in check_attend; of the ones, 2^7 each, a lane's sums are exact below 2^31 and a few are rounded, 2^-20
    assert ((lse[0].double() - torch.log(total)).abs() <= 2.0 ** -19).all()
    want = (p.T @ sv[:n, 0]) / total[:, None]
    size = (p.T @ sv[:n, 0].abs()) / total[:, None]
    # (the floor of a weight's split: 2^-31 of the largest weight, and sums over n weighted values)
    big = (0.2 * (sk[:n, 0].abs() @ q[0].double().abs().T)).max()
    tol = (4 * float(big) * (dim + 8) * 2.0 ** -23 + n * 2.0 ** -23 + 2.0 ** -18) * size + n * 2.0 ** -29 * (p / total * sv[:n, 0].abs().amax(-1)[:, None]).amax(0)[:, None]
    assert ((out[0].double() - want).abs() <= tol).all()
    cache.close()


def test_a_warp_gives_up_as_one():
    """The wait of the attention's warps: where half of the lanes give up and the others do not, all have given up.  The
    self-test reports its time-out only then."""
    import eos_b200
    rt = eos_b200.Runtime(0)
    for _ in range(3):
        with pytest.raises(eos_b200.EosB200DeviceStatusError, match="timeout"):
            rt.selftest_bounded_wait(200_000)
    s = Sequences("mx8", 64, 1, 16, [40], runtime=rt)
    s.append(*tensors(40, 1, 64, "f16", 95), [0], [40])
    s.sync()
    rt.close()


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8", "mx4"])
@pytest.mark.parametrize("top", [1e38, 1.6e38, 2.2e38])
def test_scores_as_low_as_fp32_goes(fmt, top):
    """All scores of a row close to -top, times log2(e) down to -3.2e38: the softmax is that of their differences, here none or
    more than any weight.  And both ends in one row."""
    dim, n = 32, 40
    _, v = tensors(n, 1, dim, "f16", 5)
    v = stored(v, fmt).half()
    k = torch.zeros((n, 1, dim), device="cuda", dtype=torch.float16)
    k[:, 0, 0] = -2.0
    k[[3, 37], 0, 0] = -1.0
    k[20, 0, 1] = 2.0                                      # (the second query's one large score)
    s = Sequences(fmt, dim, 1, 16, [n])
    s.append(k, v, [0], [n])
    q = torch.zeros((1, 2, dim), device="cuda")
    q[0, :, 0] = top / 2 * 2.0 ** -100                     # scores -top, and -top / 2 of tokens 3 and 37
    q[0, 1, 1] = top / 2 * 2.0 ** -100                     # token 20: 0 = -top + top
    out, lse = s.attend(q, [n], 2.0 ** 100)
    s.sync()
    two = v[[3, 37], 0].double()
    tol = (2.0 ** -14 if fmt == "bf16" else 2.0 ** -20) * two.abs().mean(0) + 2.0 ** -24 * two.abs().amax()
    assert ((out[0, 0].double() - two.mean(0)).abs() <= tol).all()
    assert abs(float(lse[0, 0]) + top / 2) <= 2.0 ** -20 * top
    assert ((out[0, 1].double() - v[20, 0].double()).abs() <= 2.0 ** -20 * v[20, 0].abs() + 2.0 ** -24).all()
    assert abs(float(lse[0, 1])) <= 2.0 ** -20 * top
    # every score the same, at the lowest
    k[:, 0, :2] = torch.tensor([-2.0, 0.0], device="cuda")
    s.append(k, v, [0], [n])
    out, lse = s.attend(q, [n], 2.0 ** 100)
    s.sync()
    mean, size = v[:, 0].double().mean(0), v[:, 0].double().abs().mean(0)
    assert ((out[0] - mean).abs() <= (n + 16) * 2.0 ** -23 * size + 2.0 ** -24).all()
    assert ((lse[0].double() + top).abs() <= 2.0 ** -20 * top).all()
    # and at the highest
    out, lse = s.attend(-q, [n], 2.0 ** 100)
    s.sync()
    assert ((out[0] - mean).abs() <= (n + 16) * 2.0 ** -23 * size + 2.0 ** -24).all()
    assert ((lse[0].double() - top).abs() <= 2.0 ** -20 * top).all()
    # a row that rises from the lowest to the highest, record by record
    k[:, 0, 0] = torch.linspace(-2, 2, 5, device="cuda").half().repeat_interleave(8)
    s.append(k, v, [0], [n])
    out, lse = s.attend(q, [n], 2.0 ** 100)
    s.sync()
    assert ((out[0] - v[32:, 0].double().mean(0)).abs() <= 24 * 2.0 ** -23 * v[32:, 0].double().abs().mean(0) + 2.0 ** -24).all()
    assert ((lse[0].double() - top).abs() <= 2.0 ** -20 * top).all()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("power", [-118, -100, 60, 100, 112, 118])
def test_keys_of_any_size_under_queries_of_the_opposite(fmt, power):
    """Block-scaled keys of 2^power under queries of 2^-power, all of one sign: the scores are of ordinary size, and so must all be
    that leads to them.  One query of the group is far smaller than the others: its scores are zeros nearly."""
    dim, n, group = 128, 70, 3
    s = Sequences(fmt, dim, 1, 16, [n])
    g = torch.Generator().manual_seed(97)
    k = (torch.rand((n, 1, dim), generator=g) * 2.0 ** power).cuda()
    v = torch.randn((n, 1, dim), generator=g).cuda()
    q = (torch.rand((1, group, dim), generator=g) * 2.0 ** -power).cuda()
    q[0, 1] *= 2.0 ** -6
    s.append(k, v, [0], [n])
    out, lse = s.attend(q, [n], 0.125)
    s.sync()
    check_attend(q, ([stored(k, fmt)], [stored(v, fmt)]), [n], 0.125, 0, fmt, out, lse, group)


def test_refusals_at_the_limits():
    """Arguments that no kernel could use: a scale that leaves fp32's range in base 2, arrays of words that are not aligned."""
    import eos_b200
    rt = eos_b200.Runtime(0)
    c = eos_b200.KvCache(rt, 4, 16, 2, 64, "mx8")
    x, i = torch.zeros((4, 2, 64), device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    p, t = x.data_ptr(), i.data_ptr()
    ok = dict(d_query=p, type="f32", q_heads=2, batch=1, d_page_table=t, max_pages=1, d_lengths=t, d_out=p + 1024, scale=1.0)
    for scale in (2.4e38, -3.4e38):
        with pytest.raises(eos_b200.EosB200Error, match="scale"):
            c.attend_device(**{**ok, "scale": scale})
    for bad in (dict(d_lse=p + 2046), dict(d_page_table=t + 1), dict(d_lengths=t + 2)):
        with pytest.raises(eos_b200.EosB200Error, match="aligned"):
            c.attend_device(**{**ok, **bad})
    rows = dict(d_key=p, d_value=p + 1024, type="f32", tokens=1, batch=1, d_page_table=t, max_pages=1, d_starts=t)
    for call in (c.append_device, c.read_device):
        for bad in (dict(d_page_table=t + 2), dict(d_starts=t + 1), dict(d_cu_tokens=t + 3)):
            with pytest.raises(eos_b200.EosB200Error, match="aligned"):
                call(**{**rows, **bad})
    c.attend_device(**{**ok, "scale": 2.3e38, "stream": torch.cuda.current_stream().cuda_stream})
    c.sync(torch.cuda.current_stream().cuda_stream)


def test_a_cache_may_outlive_its_runtime():
    """Where both are garbage of one cycle the runtime may go first; the cache then frees what it holds without looking at it,
    and leaves no error behind for the next call."""
    import ctypes

    import eos_b200
    from eos_b200 import _lib
    dim, n = 64, 40
    k, v = tensors(n, 1, dim, "f16", 101)
    for _ in range(4):
        s = Sequences("mx8", dim, 1, 16, [n])
        s.append(k, v, [0], [n])
        s.sync()
        _lib.lib().eos_b200_runtime_destroy(s.rt.handle)
        s.rt.handle = ctypes.c_void_p()
        other = Sequences("mx4", dim, 1, 16, [n])            # (takes the freed memory)
        junk = [eos_b200.Runtime(0) for _ in range(3)]
        for rt in junk:
            rt.close()
        s.cache.close()
        other.append(k, v, [0], [n])
        other.sync()
        assert same(other.read([0], [n])[0], stored(k, "mx4"))


@pytest.mark.parametrize("counts", [[100, -80, 40], [64, -64, 64], [200, -300, 150, -50], [10, -1, 0], [0, 0, 120, -120, 0, 0]])
def test_row_offsets_that_run_backwards_are_reported(counts):
    """Rows between offsets that descend belong to no one sequence; whichever of them are written or read, the call is reported,
    and what other sequences hold stays."""
    import eos_b200
    dim, heads, n = 32, 2, 208
    batch = len(counts)
    s = Sequences("mx8", dim, heads, 16, [n] * batch)
    k, v = tensors(n, heads, dim, "f16", 98)
    s.append(k, v, [0] * batch, counts)
    with pytest.raises(eos_b200.EosB200DeviceStatusError, match="row offset"):
        s.sync()
    cu = [sum(counts[:i]) for i in range(batch + 1)]
    rows = s._ints(cu), s._ints([0] * batch)
    rk, rv = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    s.cache.read_device(rk.data_ptr(), rv.data_ptr(), "f16", n, batch, s.table.data_ptr(), s.max_pages, rows[1].data_ptr(),
                        rows[0].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    with pytest.raises(eos_b200.EosB200DeviceStatusError, match="row offset"):
        s.sync()
    s.sync()
    s.append(k[:batch].contiguous(), v[:batch].contiguous(), [n - 1] * batch)     # (and the cache works on)
    s.sync()


def test_many_row_offsets():
    """More sequences than a block has threads, one of them at the end."""
    import eos_b200
    batch, n = 2000, 3
    s = Sequences("f16", 32, 1, 16, [n] * batch)
    k, v = tensors(n * batch, 1, 32, "f16", 99)
    s.append(k, v, [0] * batch, [n] * batch)
    s.sync()
    rk, rv = s.read([0] * batch, [n] * batch, "f16")
    assert same(rk, k) and same(rv, v)
    s.append(k, v, [0] * batch, [n] * (batch - 1) + [-1])
    with pytest.raises(eos_b200.EosB200DeviceStatusError, match="row offset"):
        s.sync()
    s.append(k, v, [0] * batch, [n] * (batch - 1) + [n + 1])
    with pytest.raises(eos_b200.EosB200DeviceStatusError, match="row offset"):
        s.sync()


def test_attends_that_overlapped_leave_nothing_behind():
    """Attends of one cache that no order keeps apart share its workspace, and their results are not to be used.  Those of
    calls behind them, in order again, are right: every call leaves the workspace's counts as it wants to find them."""
    dim, heads, group = 64, 2, 4
    shapes = [([20000, 3000], 0), ([20000, 3000], 700), ([1, 3000], 0), ([12000, 0], 0)]
    s = Sequences("mx8", dim, heads, 64, [20000, 3000])
    k, v = tensors(23000, heads, dim, "f16", 105)
    s.append(k, v, [0, 0], [20000, 3000])
    q = tensors(2, heads * group, dim, "f16", 106)[0]
    want = [s.attend(q, n, 0.125, window) for n, window in shapes]
    lengths = [s._ints(n) for n, _ in shapes]
    streams = [torch.cuda.Stream() for _ in shapes]
    outs = [torch.empty_like(q) for _ in shapes]
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(20):
            for (_, window), n, out, stream in zip(shapes, lengths, outs, streams):
                s.cache.attend_device(q.data_ptr(), "f16", heads * group, 2, s.table.data_ptr(), s.max_pages, n.data_ptr(),
                                      out.data_ptr(), 0.125, window, stream=stream.cuda_stream)
        torch.cuda.synchronize()
        for (n, window), (out, lse) in zip(shapes, want):
            again, lse2 = s.attend(q, n, 0.125, window)
            assert same(again, out) and same(lse2, lse)
    s.sync()


@pytest.mark.parametrize("fmt,type_,dim,group", [("bf16", "bf16", 128, 130), ("mx4", "f32", 64, 200), ("f16", "f16", 96, 70), ("mx8", "bf16", 32, 300),
                                                 ("bf16", "f32", 256, 65)])
def test_many_query_heads_over_a_sequence_that_is_cut(fmt, type_, dim, group):
    """Several chunks of query heads for a key head, the last one short, in units that tens of CTAs hold parts of: joined by
    neighbours, over the groups, and beside a short sequence."""
    lengths = [9, 13001]
    s = Sequences(fmt, dim, 1, 64, lengths, seed=4)
    k, v = tensors(sum(lengths), 1, dim, type_, 111)
    s.append(k, v, [0, 0], lengths)
    q = tensors(2, group, dim, type_, 112)[0]
    scale = 2 * dim ** -0.5
    out, lse = s.attend(q, lengths, scale)
    s.sync()
    cut = lambda x: torch.split(stored(x, fmt), lengths)  # noqa: E731
    check_attend(q, (cut(k), cut(v)), lengths, scale, 0, fmt, out, lse, group)
    again, lse2 = s.attend(q, lengths, scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("seed", range(48))
def test_shapes_at_random(seed):
    """Any format, type, head size, sharing, page and lengths: written in two calls, read back from anywhere, attended to through
    any strides and windows."""
    r = random.Random(1000 + seed)
    fmt, type_, dim = r.choice(["f16", "bf16", "mx8", "mx4"]), r.choice(["f32", "f16", "bf16"]), r.choice([32, 64, 96, 128, 192, 256])
    heads, group = r.choice([1, 2, 3, 5, 8]), r.choice([1, 2, 3, 4, 7, 8, 9, 12, 16, 17, 31, 40, 65])
    page, batch, window = r.choice([16, 32, 48, 80, 256]), r.choice([1, 2, 3, 7, 20, 60, 150]), r.choice([0, 0, 0, 1, 15, 16, 17, 100, 1000])
    most = max(1, min(4000, 200000 // (batch * heads * max(1, group // 4) * dim // 64 + 1)))
    n = [r.choice([0, 1, r.randint(0, most), int(most ** r.random()), most]) for _ in range(batch)]
    n[0] = max(n[0], 1)
    s = Sequences(fmt, dim, heads, page, n, seed=seed)
    k, v = tensors(sum(n), heads, dim, type_, seed)
    first = [r.randint(0, x) for x in n]
    at = np.cumsum([0] + n)
    rows = lambda lo, hi: np.concatenate([np.arange(at[b] + lo[b], at[b] + hi[b]) for b in range(batch)])  # noqa: E731
    for lo, hi in (([0] * batch, first), (first, n)):
        some = rows(lo, hi)
        if len(some):
            s.append(k[some].contiguous(), v[some].contiguous(), lo, [b - a for a, b in zip(lo, hi)])
    sk, sv = stored(k, fmt), stored(v, fmt)
    lo = [r.randint(0, x) for x in n]
    hi = [r.randint(a, x) for a, x in zip(lo, n)]
    rk, rv = s.read(lo, [b - a for a, b in zip(lo, hi)], fill=-3.0)
    some = rows(lo, hi)
    assert same(rk[:len(some)], sk[some]) and same(rv[:len(some)], sv[some]) and (rk[len(some):] == -3).all()
    q = tensors(batch, heads * group, dim, type_, seed + 1)[0]
    strides, view = (0, 0), q
    if r.random() < 0.5:
        head, more, off = dim + r.choice([0, 1, 8, 4]), r.choice([0, 3, 8]), r.choice([0, 1, 8])
        strides = heads * group * head + more, head
        view = torch.as_strided(torch.zeros(batch * strides[0] + 8, dtype=q.dtype, device="cuda"), q.shape, strides + (1,), off)
        view.copy_(q)
    scale = dim ** -0.5 * r.choice([1, 1, 0.1, 3, -1])
    out, lse = s.attend(view, n, scale, window, strides, shape=q.shape)
    s.sync()
    few = sorted({0, batch - 1} | {r.randrange(batch) for _ in range(3)})
    check_attend(q[few], [[x[at[b]:at[b + 1]] for b in few] for x in (sk, sv)], [n[b] for b in few], scale, window, fmt, out[few], lse[few], group)
    assert torch.isfinite(out.float()).all()
    again, lse2 = s.attend(view, n, scale, window, strides, shape=q.shape)
    assert same(out, again) and same(lse, lse2)


@pytest.mark.parametrize("fmt", ["f16", "mx8", "mx4"])
def test_attends_and_reads_while_the_next_tokens_are_appended(fmt):
    """What lies behind the length may be written while the positions before it are read: tokens of very unlike size, zeros and
    values that are not finite, at the places beside the last one and in the same words."""
    dim, heads, group, n, more = 128, 2, 4, [1001, 40], 9
    s = Sequences(fmt, dim, heads, 32, [x + more for x in n])
    k, v = tensors(sum(n), heads, dim, "f16", 121)
    s.append(k, v, [0, 0], n)
    q = tensors(2, heads * group, dim, "f16", 122)[0]
    want, lse = s.attend(q, n, 0.125)
    rk, rv = s.read([0, 0], n, "f16")
    table = []                                       # rows of `more` tokens for each sequence
    for size in (2.0 ** -14, 1.0, 2.0 ** 12, float("nan"), 0.0):
        x = tensors(2 * more, heads, dim, "f32", 123)[1] * size
        x[:, :, 32:64] *= 2.0 ** -18
        table.append(x)
    reader, writer = torch.cuda.Stream(), torch.cuda.Stream()
    cu, at, lengths, zero = s._ints([0, more, 2 * more]), s._ints(n), s._ints(n), s._ints([0, 0])
    all_cu = s._ints([0, n[0], n[0] + n[1]])
    outs = [torch.empty_like(q) for _ in range(60)]
    reads = [(torch.empty_like(rk), torch.empty_like(rv)) for _ in outs]
    torch.cuda.synchronize()
    for i, (out, (k2, v2)) in enumerate(zip(outs, reads)):
        for j in range(3):
            x = table[(3 * i + j) % len(table)]
            s.cache.append_device(x.data_ptr(), x.data_ptr(), "f32", 2 * more, 2, s.table.data_ptr(), s.max_pages, at.data_ptr(),
                                  cu.data_ptr(), stream=writer.cuda_stream)
        s.cache.attend_device(q.data_ptr(), "f16", heads * group, 2, s.table.data_ptr(), s.max_pages, lengths.data_ptr(),
                              out.data_ptr(), 0.125, stream=reader.cuda_stream)
        s.cache.read_device(k2.data_ptr(), v2.data_ptr(), "f16", sum(n), 2, s.table.data_ptr(), s.max_pages, zero.data_ptr(),
                            all_cu.data_ptr(), stream=reader.cuda_stream)
    torch.cuda.synchronize()
    for out, (k2, v2) in zip(outs, reads):
        assert same(out, want) and same(k2, rk) and same(v2, rv)
    s.sync()


def test_a_table_that_names_no_page():
    """2^27 records of two sequences, none of them on a page: nothing is attended to, and it is reported, once."""
    import eos_b200
    rt = eos_b200.Runtime(0)
    dim, page, wide = 32, 65536, 32768
    cache = eos_b200.KvCache(rt, 1, page, 1, dim, "mx4")
    table = torch.full((2, wide), -1, dtype=torch.int32, device="cuda")
    table[1, 1:] = 1
    q = tensors(2, 2, dim, "f16", 131)[0]
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    lengths = torch.tensor([2 ** 30, 2 ** 30], dtype=torch.int32, device="cuda")
    for _ in range(2):
        cache.attend_device(q.data_ptr(), "f16", 2, 2, table.data_ptr(), wide, lengths.data_ptr(), out.data_ptr(), 0.2, 0, lse.data_ptr(),
                            stream=st)
        with pytest.raises(eos_b200.EosB200DeviceStatusError, match="page"):
            cache.sync(st)
        assert (out == 0).all() and (lse == float("-inf")).all()
    cache.sync(st)
    cache.close()
