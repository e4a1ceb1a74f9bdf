"""Paged key-value cache on the device, at the limits of what its calls allow: the bits that results carry, the range of
scores and lengths, errors and workspaces of caches that live side by side."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_kv_cache import DTYPES, Sequences, stored, tensors  # noqa: E402


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
