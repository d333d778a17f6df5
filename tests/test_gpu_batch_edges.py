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
