"""Edges of the operators that decode a batch of continuations of one prompt:
values, scores and scales that are not ordinary, and what a call may be given."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import ramvamp_b200

    return ramvamp_b200


@pytest.fixture(autouse=True)
def no_device_error(rv):
    yield
    rv.device_status(0)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def caches(rv, n_seqs, cap, heads, dim, prefix, fmt, seed):
    pre, suf = rv.KvCache(1, max(prefix, 1), heads, dim, fmt), rv.KvCache(n_seqs, cap, heads, dim, fmt)
    for i, c in enumerate((pre, suf)):
        rows = (c.n_seqs, c.capacity, heads, dim)
        rv.kv_append(c, randn(seed + i, *rows), randn(seed + 2 + i, *rows) + 0.25)
    return pre, suf


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_each_sequence_keeps_its_own_mark_of_a_value_that_is_not_finite(rv, dim, dtype):
    """Many short suffixes a CTA, of which every other one holds a NaN among its
    newest tokens' values: NaN for the queries of that head that see it (in its
    column at least), the same bits as without it for all others, call after call."""
    n, Q, H, Hkv = 200, 4, 8, 4
    pre, suf = caches(rv, n, 24, Hkv, dim, 40, rv.KV_F16, 61)
    lens = [Q + (7 * b) % 21 for b in range(n)]
    q = randn(65, n, Q, H, dim).to(dtype)
    clean = rv.prefix_attention(q, pre, 40, suf, i32(lens))
    assert torch.isfinite(clean).all()
    marked = torch.zeros(n, Q, H, dtype=torch.bool, device="cuda")
    for b in range(0, n, 2):
        token, head = b // 2 % Q, b // 2 % Hkv  # one of the Q newest tokens
        suf.v[b, lens[b] - Q + token, head, b % dim] = math.nan
        marked[b, token:, head * (H // Hkv):(head + 1) * (H // Hkv)] = True
    for _ in range(20):
        got = rv.prefix_attention(q, pre, 40, suf, i32(lens))
        assert torch.equal(torch.isnan(got).any(-1), marked)
        assert torch.equal(got[~marked], clean[~marked])


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_a_query_with_a_nan_gives_nan(rv, fmt, dtype, dim):
    """All its scores are NaN, so its output row is, and no other one is touched:
    with few rows and (f16) with enough to pair two streams, with and without own
    tokens and a prefix."""
    for n, prefix in ((3, 300), (70, 300), (3, 0), (3, 2)):
        lens = [(5 * b) % 20 for b in range(n)]
        if prefix == 0:
            lens = [x + 2 for x in lens]
        pre, suf = caches(rv, n, 24, 2, dim, prefix, getattr(rv, fmt), 71)
        q = randn(75, n, 2, 8, dim).to(dtype)
        clean = rv.prefix_attention(q, pre, prefix, suf, i32(lens))
        assert torch.isfinite(clean).all()
        q[1, 0, 2, dim // 2] = math.nan
        q[2, 1, 7] = math.nan
        got = rv.prefix_attention(q, pre, prefix, suf, i32(lens))
        marked = torch.zeros(n, 2, 8, dtype=torch.bool, device="cuda")
        marked[1, 0, 2] = marked[2, 1, 7] = True
        assert torch.isnan(got[marked]).all()
        assert torch.equal(got[~marked], clean[~marked])


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_a_nan_key_gives_nan_where_it_is_all_that_a_part_sees(rv, fmt, dtype, dim):
    """A sequence's only token, a prefix's only token, the last token alone in its
    tile, and a whole tile of them: every row that sees one is NaN, the others keep
    their bits.  An 8-bit row that held an infinity counts as NaN."""
    fmt = getattr(rv, fmt)
    bad = math.nan if fmt == rv.KV_F16 else math.inf  # as appended

    def run(prefix, lens, spoil, n_q=1):
        pre, suf = caches(rv, len(lens), 300, 2, dim, prefix, fmt, 81)
        q = randn(85, len(lens), n_q, 8, dim).to(dtype)
        clean = rv.prefix_attention(q, pre, prefix, suf, i32(lens))
        spoil(pre, suf)
        return clean, rv.prefix_attention(q, pre, prefix, suf, i32(lens))

    def spoil(cache, seq, head, positions):  # the first value of a key row, through kv_append
        k, v = rv.kv_read(cache, cache.capacity)
        keep = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
        k[seq, positions, head, 0] = bad
        rv.kv_append(cache, k, v)
        for t, old in zip([t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None], keep):
            new = t[seq, positions, head].clone()  # nothing else changes by a rounding
            t.copy_(old)
            t[seq, positions, head] = new

    # one sequence's only token, of kv head 1
    clean, got = run(200, [1, 1, 40], lambda pre, suf: spoil(suf, 1, 1, [0]))
    assert torch.isnan(got[1, :, 4:]).all()
    got[1, :, 4:] = clean[1, :, 4:]
    assert torch.equal(got, clean)
    # the same without a prefix, and the first of two queries sees nothing
    clean, got = run(0, [1, 9], lambda pre, suf: spoil(suf, 0, 0, [0]), n_q=2)
    assert not got[0, 0].any() and torch.isnan(got[0, 1, :4]).all()
    got[0, 1, :4] = clean[0, 1, :4]
    assert torch.equal(got, clean)
    # the prefix's only token
    clean, got = run(1, [5, 0, 130], lambda pre, suf: spoil(pre, 0, 0, [0]))
    assert torch.isnan(got[:, :, :4]).all() and torch.equal(got[:, :, 4:], clean[:, :, 4:])
    # the last token of 129, in a tile of its own, of the prefix and of a suffix
    clean, got = run(129, [5, 0, 130], lambda pre, suf: spoil(pre, 0, 0, [128]))
    assert torch.isnan(got[:, :, :4]).all() and torch.equal(got[:, :, 4:], clean[:, :, 4:])
    clean, got = run(0, [5, 129, 130], lambda pre, suf: spoil(suf, 1, 0, [128]))
    assert torch.isnan(got[1, :, :4]).all()
    got[1, :, :4] = clean[1, :, :4]
    assert torch.equal(got, clean)
    # a whole tile of a long prefix
    clean, got = run(3000, [5, 0, 130], lambda pre, suf: spoil(pre, 0, 1, list(range(1024, 1152))))
    assert torch.isnan(got[:, :, 4:]).all() and torch.equal(got[:, :, :4], clean[:, :, :4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("factor", [2.0 ** 12, 2.0 ** 24, 2.0 ** 40, 2.0 ** 90])
def test_8_bit_values_of_later_tokens_do_not_reach_earlier_queries(rv, dtype, dim, factor):
    """Of five new tokens the fourth has finite values far larger than the
    others': the first three queries keep their bits."""
    for length in (5, 126, 131, 260):
        pre, suf = caches(rv, 2, 300, 2, dim, 130, rv.KV_Q8, 91)
        q = randn(95, 2, 5, 8, dim).to(dtype)
        clean = rv.prefix_attention(q, pre, 130, suf, i32([300, length]))
        suf.v_scale[1, length - 2] *= factor
        got = rv.prefix_attention(q, pre, 130, suf, i32([300, length]))
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :3], clean[1, :3])
        assert not torch.equal(got[1, 3:], clean[1, 3:])


def attention_by_weight(q, pre, prefix_len, suf, lens, scale):
    """(output, bound of the error) in 64 bits, one query token a sequence.

    A score is off by at most delta_j = 2^-20 scale max|q| sum|k_j| (f32 sums of
    at most 256 products: 2^-24 each, 16 of them allowed for), so a weight by
    eps_j = 2 delta_j + 2^-19 of itself (exponential, running rescales), and by
    2^-11 more where it is rounded to f16.  That moves the output by at most
    sum p_j eps_j |v_j| + (sum p_j eps_j) sum p_j |v_j|.  Products of weight and
    value scale below 2^-14, where the row's largest is 2^5 or more, are held
    within 2^-25: 2^-30 of the largest product a key.  An f16 output is rounded
    (2^-11 of it)."""
    f16 = q.dtype == torch.float16
    values = lambda c: [x.double() * s.double().unsqueeze(-1) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]  # noqa: E731
    (pk, pv), (sk, sv) = values(pre), values(suf)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    G = q.shape[2] // pre.n_kv_heads
    for b, n in enumerate(lens):
        k, v = (torch.cat([p[0, :prefix_len], s[b, :n]]).repeat_interleave(G, 1) for p, s in ((pk, sk), (pv, sv)))
        qq = q[b, 0].double()
        p = torch.softmax(torch.einsum("hd,khd->hk", qq, k) * scale, -1)
        eps = 2 * 2.0 ** -20 * scale * qq.abs().amax(-1)[:, None] * k.abs().sum(-1).t() + 2.0 ** -19 + f16 * 2.0 ** -11
        size = torch.einsum("hk,khd->hd", p, v.abs())
        out[b, 0] = torch.einsum("hk,khd->hd", p, v)
        tol[b, 0] = torch.einsum("hk,khd->hd", p * eps, v.abs()) + (p * eps).sum(-1)[:, None] * size
        tol[b, 0] += (len(k) * 2.0 ** -30 * (p * v.abs().amax(-1).t()).amax(-1))[:, None] + f16 * 2.0 ** -11 * out[b, 0].abs()
    return out, tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_8_bit_values_count_by_their_weight(rv, dtype, dim):
    """Values far larger than the others' on keys that weigh next to nothing,
    and sizes spread over many powers of two: the error is bounded by weight
    times value, not by the largest value."""
    n, prefix, lens = 3, 700, [1, 260, 129]
    scale = dim ** -0.5
    for factor in (2.0 ** 12, 2.0 ** 24, 2.0 ** 40, None):
        pre, suf = caches(rv, n, 260, 2, dim, prefix, rv.KV_Q8, 101)
        q = randn(105, n, 1, 8, dim)
        q = (0.2 * q + q[:, :, :, :1].sign().expand_as(q)).to(dtype)  # all near + or - (1, .., 1)
        q = q.abs()
        if factor:
            for cache, seq, at in ((pre, 0, 3), (pre, 0, 400), (suf, 1, 200), (suf, 2, 0)):
                k = torch.full((1, 1, 2, dim), -100 / (scale * dim), device="cuda")  # a score of about -100
                one = rv.KvCache(1, 1, 2, dim, rv.KV_Q8)
                rv.kv_append(one, k, k)
                cache.k[seq, at], cache.k_scale[seq, at] = one.k[0, 0], one.k_scale[0, 0]
                cache.v_scale[seq, at] *= factor
        else:
            for cache, seed in ((pre, 106), (suf, 107)):
                cache.v_scale *= torch.exp2(8 * randn(seed, *cache.v_scale.shape))
        got = rv.prefix_attention(q, pre, prefix, suf, i32(lens), scale=scale)
        want, tol = attention_by_weight(q, pre, prefix, suf, lens, scale)
        if dtype == torch.float16 and factor is None:
            fits = want.abs() < 60000
            got, want, tol = got[fits], want[fits], tol[fits]
            assert fits.double().mean() > 0.25
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= tol).all()


def test_sample_draws_many_from_one_row(rv):
    """An expanded row (stride 0) as a copy of it in every row."""
    logits = 2 * randn(111, 1, 5003)
    u = torch.rand(40, device="cuda", generator=gen(112))
    k = i32([50] * 40)
    tokens, logprobs = rv.sample(logits.expand(40, -1), u, top_k=k)
    want = rv.sample(logits.expand(40, -1).contiguous(), u, top_k=k)
    assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
    assert len(set(tokens.tolist())) > 1


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_a_suffix_without_room_leaves_the_prefix(rv, fmt, dtype, dim):
    """A suffix cache of capacity 0 (tensors without memory): attention over the
    prefix alone, as with an empty suffix; a length above 0 is reported."""
    fmt = getattr(rv, fmt)
    pre, one = caches(rv, 3, 1, 2, dim, 9000, fmt, 121)  # long enough for both to fill the GPU
    none = rv.KvCache(3, 0, 2, dim, fmt)
    q = randn(125, 3, 2, 8, dim).to(dtype)
    zero = i32([0, 0, 0])
    want = rv.prefix_attention(q, pre, 9000, one, zero)
    assert torch.isfinite(want).all() and want.any()
    assert torch.equal(rv.prefix_attention(q, pre, 9000, none, zero), want)
    assert not rv.prefix_attention(q, None, 0, none, zero).any()
    rv.device_status(0)
    assert torch.equal(rv.prefix_attention(q, pre, 9000, none, i32([0, 1, 0])), want)
    with pytest.raises(rv.KernelError) as e:
        rv.device_status(0)
    assert e.value.kind == "CapacityExceeded"


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("factor", [1e34, 1e36])
def test_f32_queries_near_the_end_of_their_range_over_8_bit_rows(rv, dim, factor):
    """The attention scale brings the scores back: products of queries and
    levels must not overflow before it is applied."""
    n, prefix, lens = 2, 300, [40, 7]
    pre, suf = caches(rv, n, 40, 1, dim, prefix, rv.KV_Q8, 131)
    q = randn(135, n, 1, 8, dim) * factor
    scale = dim ** -0.5 / factor
    got = rv.prefix_attention(q, pre, prefix, suf, i32(lens), scale=scale)
    want, tol = attention_by_weight(q, pre, prefix, suf, lens, scale)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("factor", [1e-32, 1e-36])
def test_f32_queries_near_the_small_end_of_their_range(rv, fmt, dim, factor):
    """Queries below 2^-100 keep their bits: times a power of two they give what
    ordinary ones do."""
    n, prefix, lens = 2, 300, [40, 7]
    pre, suf = caches(rv, n, 40, 1, dim, prefix, getattr(rv, fmt), 141)
    q = randn(145, n, 1, 8, dim)
    two = 2.0 ** round(math.log2(factor))
    want = rv.prefix_attention(q, pre, prefix, suf, i32(lens), scale=dim ** -0.5)
    got = rv.prefix_attention(q * two, pre, prefix, suf, i32(lens), scale=dim ** -0.5 / two)
    # the same products, but for values of q * two below 2^-126 that lose bits
    assert (got - want).abs().max() <= 2.0 ** -18 * want.abs().max()


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_f32_sums_over_a_long_prompt(rv, fmt, dim):
    """So many rows that a stream runs through hundreds of tiles of one segment,
    values of one sign, weights nearly alike.  Within 512 keys the products are
    summed by the tensor cores: 64 additions that lose less than 2^-23 of the sum
    each, 2^-17; sums of these are f32 (at most 128 of them: 2^-17 at worst).  The
    weights are off by 2 delta_j + 2^-19 as above."""
    n, Q, H, prefix = 128, 16, 8, 32768
    pre, suf = caches(rv, n, 16, 1, dim, prefix, getattr(rv, fmt), 151)
    pre.v.abs_()
    suf.v.abs_()
    q = 0.02 * randn(155, n, Q, H, dim)
    got = rv.prefix_attention(q, pre, prefix, suf, i32([Q] * n))
    value = lambda x, s: x.double() if s is None else x.double() * s.double().unsqueeze(-1)  # noqa: E731
    for b in (0, 77):
        k = torch.cat([value(pre.k, pre.k_scale)[0], value(suf.k, suf.k_scale)[b]])[:, 0]
        v = torch.cat([value(pre.v, pre.v_scale)[0], value(suf.v, suf.v_scale)[b]])[:, 0]
        s = q[b].double() @ k.t() * dim ** -0.5
        s.masked_fill_(torch.arange(len(k), device="cuda") > prefix + torch.arange(Q, device="cuda")[:, None, None], -math.inf)
        p = torch.softmax(s, -1)
        eps = 2 * 2.0 ** -20 * dim ** -0.5 * q[b].double().abs().amax(-1, keepdim=True) * k.abs().sum(-1) + 2.0 ** -19
        want = p @ v  # all terms are positive: the sums of their sizes, too
        tol = (p * eps) @ v + (p * eps).sum(-1, keepdim=True) * want + 2.0 ** -16 * want
        assert ((got[b].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
def test_f32_sums_over_a_long_prompt_repeat_bit_for_bit(rv, fmt):
    """A row's runs are added in memory by one thread, in order."""
    pre, suf = caches(rv, 128, 16, 1, 128, 32768, getattr(rv, fmt), 161)
    q = randn(165, 128, 8, 8, 128)
    lens = i32([8 + b % 9 for b in range(128)])
    first = rv.prefix_attention(q, pre, 32768, suf, lens)
    assert torch.isfinite(first).all()
    for _ in range(10):
        assert torch.equal(rv.prefix_attention(q, pre, 32768, suf, lens), first)
