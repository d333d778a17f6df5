"""The operators that decode a batch of continuations of one prompt -- KV cache
rows in f16 and 8 bits, attention over a shared prefix, sampling -- against
plain implementations in 64 bits (numpy / torch on the CPU or the GPU)."""
import math

import numpy as np
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


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device="cuda")


# ------------------------------------------------------------------ KV cache
def q8_rows(x):
    """Levels and scales by the format's definition, in numpy f32 (one IEEE
    rounding an operation, so the kernel's must be the same bits)."""
    x = x.astype(np.float32)
    amax = np.abs(x).max(-1, keepdims=True)  # NaN propagates
    zero = amax < np.float32(2.0 ** -50)
    with np.errstate(all="ignore"):
        inv = np.where(zero, np.float32(0), np.float32(1) / amax * np.float32(127))
        lv = np.rint(x * inv)
        lv = np.where(np.isnan(lv), 0, lv)
    return lv.astype(np.int8), np.where(zero, np.float32(0), amax * (np.float32(1) / np.float32(127)))[..., 0]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,dim", [(4, 128), (8, 64), (1, 8), (3, 80), (5, 256)])
def test_kv_q8_levels_and_scales_are_exact(rv, dtype, heads, dim):
    n_seqs, n, cap = 3, 7, 40
    g = gen(dim + heads)
    x = torch.randn(2, n_seqs, n, heads, dim, device="cuda", generator=g).to(getattr(torch, dtype))
    x[0, 0, 0, 0] = 0                       # a zero row
    x[1, 1, 2, 0] = x[1, 1, 2, 0] * 1e-16   # below 2^-50 in f32 and bf16, zero in f16
    x[0, 2, 1, 0, 0] = math.inf             # reads back as NaN
    x[1, 2, 3, 0, dim - 1] = math.nan
    cache = rv.KvCache(n_seqs, cap, heads, dim, rv.KV_Q8)
    lens = i32([n, 20, cap])
    rv.kv_append(cache, x[0], x[1], lens=lens)
    for plane, scales, rows in ((cache.k, cache.k_scale, x[0]), (cache.v, cache.v_scale, x[1])):
        lv, sc = q8_rows(rows.float().cpu().numpy())
        for b, end in enumerate(lens.tolist()):
            assert np.array_equal(plane[b, end - n:end].cpu().numpy(), lv[b])
            assert np.array_equal(scales[b, end - n:end].cpu().numpy(), sc[b], equal_nan=True)
            assert not plane[b, :end - n].any() and not plane[b, end:].any()  # nothing else written
    k, v = rv.kv_read(cache, n, lens=lens)
    for back, rows in ((k, x[0]), (v, x[1])):
        lv, sc = q8_rows(rows.float().cpu().numpy())
        with np.errstate(all="ignore"):
            want = lv.astype(np.float32) * sc[..., None]
        assert np.array_equal(back.cpu().numpy(), want, equal_nan=True)
    # The error of a finite row is at most half a level, up to f32 rounding.
    err = (k[0].double() - x[0, 0].double()).abs()
    assert (err <= x[0, 0].double().abs().amax(-1, keepdim=True) / 254 * (1 + 1e-5)).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_kv_f16_round_trip(rv, dtype):
    g = gen(3)
    x = (torch.randn(2, 2, 5, 4, 64, device="cuda", generator=g) * 3).to(getattr(torch, dtype))
    cache = rv.KvCache(2, 9, 4, 64, rv.KV_F16)
    rv.kv_append(cache, x[0], x[1], position=3)
    assert torch.equal(cache.k[:, 3:8], x[0].half()) and torch.equal(cache.v[:, 3:8], x[1].half())
    assert not cache.k[:, :3].any() and not cache.k[:, 8:].any()
    for out in (torch.float32, torch.float16, torch.bfloat16):
        k, v = rv.kv_read(cache, 5, position=3, dtype=out)
        assert torch.equal(k, x[0].half().to(out)) and torch.equal(v, x[1].half().to(out))


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_kv_append_from_fused_rows_of_any_alignment(rv, dtype, offset):
    """k and v inside the rows of a fused projection, at element offsets that
    are not 16-byte aligned, and a sequence shorter than the new rows."""
    n_seqs, n, H, D = 4, 3, 2, 128
    wide = torch.randn(n_seqs, n, offset + 5 * H * D + 1, device="cuda", generator=gen(offset)).to(dtype)
    k = wide[..., offset:offset + H * D].unflatten(2, (H, D))
    v = wide[..., offset + H * D:offset + 2 * H * D].unflatten(2, (H, D))
    for fmt in (rv.KV_F16, rv.KV_Q8):
        got, want = rv.KvCache(n_seqs, 8, H, D, fmt), rv.KvCache(n_seqs, 8, H, D, fmt)
        lens = i32([3, 8, 2, 0])  # the third lacks a position for its first row, the last for all
        rv.kv_append(got, k, v, lens=lens)
        rv.kv_append(want, k.contiguous(), v.contiguous(), lens=lens)
        assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v)
        assert got.k[1, 5:].any() and got.k[2, :2].any() and not got.k[2, 2:].any() and not got.k[3].any()
        kk, vv = rv.kv_read(got, n, lens=lens)
        assert not kk[2, 0].any() and not kk[3].any() and kk[2, 1].any() and not vv[3].any()


def test_kv_length_past_the_cache(rv):
    cache = rv.KvCache(2, 4, 1, 64, rv.KV_Q8)
    x = torch.ones(2, 2, 1, 64, device="cuda")
    rv.kv_append(cache, x, x, lens=i32([4, 5]))
    with pytest.raises(rv.KernelError) as e:
        rv.device_status(0)
    assert e.value.kind == "CapacityExceeded"
    assert cache.k[0, 2:].all() and cache.k[1, 3].all() and not cache.k[1, :3].any()


def test_kv_offsets_past_32_bits(rv):
    """Rows more than 2^32 bytes into a cache, written, read and attended."""
    H, D, cap = 8, 128, (1 << 32) // (8 * 128) + 300
    cache = rv.KvCache(1, cap, H, D, rv.KV_Q8)
    x = torch.randn(1, 200, H, D, device="cuda", generator=gen(9))
    rv.kv_append(cache, x, -x, position=cap - 200)
    lv, sc = q8_rows(x.cpu().numpy())
    assert np.array_equal(cache.k[0, cap - 200:].cpu().numpy(), lv[0])
    k, v = rv.kv_read(cache, 200, position=cap - 200)
    assert torch.equal(k, -v) and np.array_equal(k.cpu().numpy(), lv.astype(np.float32) * sc[..., None])
    # 2^32 bytes in, only the last 200 keys are not zero: with a large score they are all that is seen.
    q = x[:, -1:].contiguous() * 64
    none = rv.KvCache(1, 1, H, D, rv.KV_Q8)
    out = rv.prefix_attention(q, cache, cap, none, i32([0]))
    s = torch.einsum("qhd,khd->hk", q[0].double(), k[0].double()) * D ** -0.5
    assert float(s.amax(-1).min()) > 200  # the zero keys weigh less than e^-200 each
    want = torch.einsum("hk,khd->hd", torch.softmax(s, -1), v[0].double())
    assert (out[0, 0].double() - want).abs().max() < 1e-3 * float(v.abs().max())


# ---------------------------------------------------------------- attention
def cache_values(cache):
    """(k, v) in 64 bits."""
    k, v = cache.k.double(), cache.v.double()
    if cache.k_scale is not None:
        k, v = k * cache.k_scale.double().unsqueeze(-1), v * cache.v_scale.double().unsqueeze(-1)
    return k, v


def attention_64(q, prefix, prefix_len, suffix, lens, scale):
    """(output, per-row bound of the kernel's error) in 64 bits.

    The bound: scores are sums of head_dim products in f32, of queries held to
    2^-22 of the row's largest value, so a score is off by at most
    delta = 2^-20 * scale * max|q| * sum|k| (sums and products of at most 256
    terms: 2^-24 each, most of them cancelling; 16 of them are allowed for).  A
    relative error of every weight of at most 2 delta + 2^-19 (exponential,
    running rescales) moves a mean of values by at most that times twice the
    largest |v|.  f16 queries: weights may be rounded to f16 (2^-11), and the
    output is (2^-11)."""
    n, Q, H, D = q.shape
    G = H // suffix.n_kv_heads
    out = torch.zeros(n, Q, H, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros(n, Q, H, 1, dtype=torch.float64, device="cuda")
    sk, sv = cache_values(suffix)
    if prefix_len:
        pk, pv = (x[0, :prefix_len] for x in cache_values(prefix))
    for b, L in enumerate(lens):
        for i in range(Q):
            seen = max(0, L - Q + 1 + i)
            k, v = sk[b, :seen], sv[b, :seen]
            if prefix_len:
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
            if len(k) == 0:
                continue
            k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
            qq = q[b, i].double()
            p = torch.softmax(torch.einsum("hd,khd->hk", qq, k) * scale, -1)
            out[b, i] = torch.einsum("hk,khd->hd", p, v)
            delta = 2.0 ** -20 * scale * qq.abs().amax(-1) * k.abs().sum(-1).amax(0)
            vmax = v.abs().amax((0, 2))
            tol[b, i] = (2 * vmax * (2 * delta + 2.0 ** -19))[:, None]
            if q.dtype == torch.float16:
                tol[b, i] += (2.0 ** -10 * vmax)[:, None]
    return out, tol


def make_caches(rv, n_seqs, cap, Hkv, D, prefix, fmt, seed, size=1.0):
    g = gen(seed)
    pre = rv.KvCache(1, max(prefix, 1), Hkv, D, fmt)
    suf = rv.KvCache(n_seqs, cap, Hkv, D, fmt)
    for c, n in ((pre, pre.capacity), (suf, cap)):
        k = torch.randn(c.n_seqs, n, Hkv, D, device="cuda", generator=g) * size
        v = torch.randn(c.n_seqs, n, Hkv, D, device="cuda", generator=g) + 0.25
        rv.kv_append(c, k, v, position=0)
    return pre, suf


def check_attention(rv, q, pre, prefix_len, suf, lens, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    got = rv.prefix_attention(q, pre, prefix_len, suf, i32(lens), scale=scale)
    assert got.dtype == q.dtype
    want, tol = attention_64(q, pre, prefix_len, suf, lens, scale)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"largest excess {float((off / tol.clamp(min=1e-300)).max()):.3g} of the bound"
    return got


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 8, 96, 256])
def test_attention_lengths(rv, fmt, dtype, dim):
    """Prefixes and suffixes that end at, before and after a tile of keys,
    an empty prefix, empty suffixes and rows that see nothing."""
    fmt = getattr(rv, fmt)
    Hkv, G, cap = 2, 4, 300
    for prefix in (0, 1, 63, 127, 128, 129, 255, 577):
        lens = [0, 1, 2, 127, 128, 129, 300]
        pre, suf = make_caches(rv, len(lens), cap, Hkv, dim, prefix, fmt, prefix + dim)
        q = torch.randn(len(lens), 1, Hkv * G, dim, device="cuda", generator=gen(prefix)).to(dtype)
        got = check_attention(rv, q, pre, prefix, suf, lens)
        if prefix == 0:
            assert not got[0].any()
            none = rv.prefix_attention(q, None, 0, suf, i32(lens))
            assert torch.equal(none, got)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 128), (4, 4, 128), (12, 4, 64), (7, 1, 64), (40, 1, 128), (6, 2, 96)])
@pytest.mark.parametrize("n_seqs,n_q", [(1, 1), (3, 5), (17, 1), (70, 2), (2, 40)])
def test_attention_head_layouts_and_query_counts(rv, heads, kv_heads, dim, n_seqs, n_q):
    """From one query row to several row tiles, new tokens that see only the
    earlier ones, and lengths shorter than the queries (rows before a
    sequence's first token see the prefix alone)."""
    cap, prefix = 150, 333
    lens = [(n_q - 2 + 37 * b) % (cap + 1) for b in range(n_seqs)]
    lens = [max(0, x) for x in lens]
    for fmt, dtype in ((rv.KV_F16, torch.float32), (rv.KV_Q8, torch.float16), (rv.KV_Q8, torch.float32)):
        pre, suf = make_caches(rv, n_seqs, cap, kv_heads, dim, prefix, fmt, heads + n_seqs)
        q = torch.randn(n_seqs, n_q, heads, dim, device="cuda", generator=gen(n_q)).to(dtype)
        check_attention(rv, q, pre, prefix, suf, lens)
    if n_q > 1:  # no prefix: rows with nothing to see are zeros
        got = check_attention(rv, q, None, 0, suf, [min(x, n_q - 1) for x in lens])
        assert not got[:, 0].any()


@pytest.mark.parametrize("prefix", [5000, 20001])
@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
def test_attention_long_prefix_split_over_the_device(rv, prefix, fmt):
    pre, suf = make_caches(rv, 9, 700, 2, 128, prefix, getattr(rv, fmt), 1)
    lens = [1, 700, 350, 0, 3, 128, 256, 699, 64]
    for dtype in (torch.float32, torch.float16):
        q = 2 * torch.randn(9, 1, 16, 128, device="cuda", generator=gen(2)).to(dtype)
        check_attention(rv, q, pre, prefix, suf, lens)


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_attention_nothing_of_hidden_places_is_seen(rv, fmt, dim):
    """Infinities and NaN past every length, in other sequences' rows and past
    the prefix: the output is the same bits as with zeros there."""
    fmt = getattr(rv, fmt)
    lens, prefix = [0, 5, 130, 64], 200
    pre, suf = make_caches(rv, 4, 200, 2, dim, 512, fmt, 5)
    q = torch.randn(4, 3, 8, dim, device="cuda", generator=gen(6))
    outs = []
    for fill in (0.0, math.nan, math.inf, -math.inf):
        for c, ends in ((pre, [prefix]), (suf, lens)):
            for b, end in enumerate(ends):
                planes = (c.k, c.v) if fmt == rv.KV_F16 else (c.k_scale, c.v_scale)
                for plane in planes:
                    plane[b, end:] = fill
        for dtype in (torch.float32, torch.float16):
            outs.append(rv.prefix_attention(q.to(dtype), pre, prefix, suf, i32(lens)))
    assert all(torch.isfinite(o).all() for o in outs)
    assert all(torch.equal(outs[i], outs[i % 2]) for i in range(2, 8))


def test_attention_values_that_are_not_finite_reach_their_rows_only(rv):
    """A NaN value row is seen by the sequence that owns it and by no other;
    in the prefix everyone sees it."""
    pre, suf = make_caches(rv, 3, 100, 2, 128, 150, rv.KV_F16, 7)
    q = torch.randn(3, 1, 8, 128, device="cuda", generator=gen(8))
    suf.v[1, 20, 0] = math.nan
    out = rv.prefix_attention(q, pre, 150, suf, i32([100, 100, 15]))
    assert torch.isnan(out[1, 0, :4]).all() and torch.isfinite(out[1, 0, 4:]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
    pre.v[0, 149, 1] = math.inf
    out = rv.prefix_attention(q, pre, 150, suf, i32([100, 10, 15]))
    assert torch.isfinite(out[:, :, :4]).all() and not torch.isfinite(out[:, :, 4:]).any()


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_Q8"])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_later_tokens_do_not_reach_earlier_queries(rv, fmt, dim, bad):
    """Of five new tokens the fourth has a value (then a key) that is not
    finite: the first three queries are the same bits as without it, the last
    two are not finite (but for a key of infinite scale, whose scores may be
    -infinity: then it weighs nothing)."""
    fmt = getattr(rv, fmt)
    for length in (5, 126, 131, 260):
        outs = []
        for where in (None, "v", "k"):
            pre, suf = make_caches(rv, 2, 300, 2, dim, 130, fmt, 51)
            if where:
                planes = (getattr(suf, where) if fmt == rv.KV_F16 else getattr(suf, where + "_scale"))
                planes[1, length - 2] = bad
            q = torch.randn(2, 5, 8, dim, device="cuda", generator=gen(52))
            outs.append([rv.prefix_attention(q.to(t), pre, 130, suf, i32([300, length])) for t in (torch.float32, torch.float16)])
        for where, with_bad in zip("vk", outs[1:]):
            for clean, got in zip(outs[0], with_bad):
                assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :3], clean[1, :3])
                if where == "v" or fmt == rv.KV_F16 or math.isnan(bad):
                    assert not torch.isfinite(got[1, 3:]).all(-1).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_large_scores_and_sinks(rv, dim, dtype):
    """Scores that grow along the keys (the running maximum moves at every
    tile), one key that takes nearly all the weight, keys that differ by more
    than the exponent's range, values of very unequal size per token."""
    for fmt in (rv.KV_F16, rv.KV_Q8):
        pre, suf = make_caches(rv, 3, 260, 2, dim, 900, fmt, 11)
        g = gen(12)
        q = torch.randn(3, 1, 4, dim, device="cuda", generator=g).to(dtype)
        ramp = torch.linspace(0, 3, 900, device="cuda")[None, :, None, None] * torch.sign(q[0, 0, 0].float())
        k = 0.3 * torch.randn(1, 900, 2, dim, device="cuda", generator=g) + ramp
        v = torch.randn(1, 900, 2, dim, device="cuda", generator=g)
        v = v * torch.exp(3 * torch.randn(1, 900, 2, 1, device="cuda", generator=g)).clamp(max=100)
        v[0, 3] = 0  # a sink: the largest score of the first tile, no value
        k[0, 3] = 4 * torch.sign(q[1, 0, 0].float())
        rv.kv_append(pre, k, v)
        check_attention(rv, q, pre, 900, suf, [1, 260, 129])
        check_attention(rv, 20 * q, pre, 900, suf, [1, 260, 129], scale=0.5)


def test_attention_tiny_and_huge_queries_and_values(rv):
    """f32 queries outside f16's range and values near its ends."""
    for fmt in (rv.KV_F16, rv.KV_Q8):
        pre, suf = make_caches(rv, 2, 40, 1, 128, 300, fmt, 13)
        base = torch.randn(2, 1, 8, 128, device="cuda", generator=gen(14))
        for factor in (1e-30, 1e-6, 1e6, 1e20):
            check_attention(rv, base * factor, pre, 300, suf, [40, 7], scale=128 ** -0.5 / factor)
        check_attention(rv, torch.zeros_like(base), pre, 300, suf, [40, 7])
    for size in (1e-4, 400.0):
        pre, suf = make_caches(rv, 2, 40, 1, 128, 300, rv.KV_Q8, 15)
        v = size * torch.randn(1, 300, 1, 128, device="cuda", generator=gen(16))
        rv.kv_append(pre, torch.randn(1, 300, 1, 128, device="cuda", generator=gen(17)), v)
        check_attention(rv, base, pre, 300, suf, [0, 0])
        check_attention(rv, base.half(), pre, 300, suf, [0, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_strided_queries_and_given_buffers(rv, dtype):
    """Queries cut out of a fused projection (token and sequence strides, an
    odd element offset), out and scratch passed in, another stream."""
    B, Q, H, D = 5, 3, 8, 128
    pre, suf = make_caches(rv, B, 90, 2, D, 200, rv.KV_F16, 21)
    lens = [3, 90, 40, 0, 1]
    for offset in (0, 1, 8):
        wide = torch.randn(B + 1, Q + 2, offset + 2 * H * D + 3, device="cuda", generator=gen(offset)).to(dtype)
        q = wide[1:, 1:-1, offset:offset + H * D].unflatten(2, (H, D))
        want = check_attention(rv, q.contiguous(), pre, 200, suf, lens)
        out = torch.full_like(want, math.nan)
        scratch = torch.empty(rv.prefix_attention_scratch(B, Q, H, 2, D) + 64, dtype=torch.uint8, device="cuda")
        scratch.fill_(255)  # whatever it held before
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = rv.prefix_attention(q, pre, 200, suf, i32(lens), out=out, scratch=scratch)
        torch.cuda.current_stream().wait_stream(side)
        assert got is out and torch.equal(out, want)


def test_attention_repeats_bit_for_bit_and_in_a_graph(rv):
    """The same inputs give the same bits, call after call and replayed from a
    CUDA graph with other lengths in the same device array."""
    pre, suf = make_caches(rv, 6, 600, 4, 128, 3000, rv.KV_Q8, 23)
    q = torch.randn(6, 1, 32, 128, device="cuda", generator=gen(24))
    lens = i32([1, 600, 300, 20, 0, 128])
    out = torch.empty_like(q)
    scratch = torch.empty(rv.prefix_attention_scratch(6, 1, 32, 4, 128), dtype=torch.uint8, device="cuda")
    call = lambda: rv.prefix_attention(q, pre, 3000, suf, lens, out=out, scratch=scratch)  # noqa: E731
    first = call().clone()
    for _ in range(5):
        assert torch.equal(call(), first)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call()
    out.zero_()
    graph.replay()
    assert torch.equal(out, first)
    lens.copy_(i32([5, 0, 600, 599, 257, 129]))
    graph.replay()
    replayed = out.clone()
    assert torch.equal(call(), replayed)


def test_attention_over_an_engines_cache(rv):
    """One layer of an AttnEngine as the prefix, without a copy."""
    eng = rv.AttnEngine(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, max_positions=64)
    g = gen(31)
    ones = torch.ones(128, device="cuda")
    for pos in range(40):
        for layer in range(2):
            x = torch.randn(8 * 128 + 2 * 256, device="cuda", generator=g)
            eng.decode(layer, pos, x[:1024].contiguous(), x[1024:1280].contiguous(), x[1280:].contiguous(), ones, ones)
    pre = rv.KvCache.of_engine(eng, 1)
    k, v = eng.cache_tensors(1)
    same = rv.KvCache.of(k.view(torch.float16).view(1, 40, 2, 128), v.view(torch.float16).view(1, 40, 2, 128))
    _, suf = make_caches(rv, 2, 8, 2, 128, 1, rv.KV_F16, 32)
    q = torch.randn(2, 1, 8, 128, device="cuda", generator=g)
    got = rv.prefix_attention(q, pre, 40, suf, i32([8, 3]))
    assert torch.equal(got, check_attention(rv, q, same, 40, suf, [8, 3]))
    eng.close()


def test_attention_length_outside_the_cache_is_held_inside(rv):
    pre, suf = make_caches(rv, 2, 30, 2, 128, 50, rv.KV_F16, 33)
    q = torch.randn(2, 1, 4, 128, device="cuda", generator=gen(34))
    got = rv.prefix_attention(q, pre, 50, suf, i32([31, -1]))
    with pytest.raises(rv.KernelError) as e:
        rv.device_status(0)
    assert e.value.kind == "CapacityExceeded"
    assert torch.equal(got, rv.prefix_attention(q, pre, 50, suf, i32([30, 0])))


# ----------------------------------------------------------------- sampling
def kept_64(l, T, k, p, mp):
    """(token ids kept in order, their shares) in 64 bits; l: numpy f32."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float64)
    order = np.lexsort((np.arange(len(l)), -l))
    top = l[order[0]]
    with np.errstate(all="ignore"):
        w = np.where(l == top, 1.0, np.exp((l - top) / T))[order]
    w = np.where(np.isnan(w), 0.0, w)
    keep = len(l) if k <= 0 or k >= len(l) else k
    if p < 1:
        before = np.cumsum(w[:keep]) - w[:keep]
        keep = max(1, int((before < p * w[:keep].sum()).sum()))
    keep = max(1, int((w[:keep] >= mp).sum()))
    return order[:keep], w[:keep] / w[:keep].sum()


def middle_u(l, T, k, p, mp, rng, draws, least=1e-5):
    """u in the middle of random kept tokens' intervals (tokens of share above
    `least`, far wider than the 1e-6 that f32 exponentials may move an edge):
    (u, token, ln share)."""
    ids, share = kept_64(l, T, k, p, mp)
    by_index = np.argsort(ids)
    edges = np.cumsum(share[by_index])
    able = np.flatnonzero(share[by_index] > least)
    picks = rng.choice(able, size=draws)
    u = edges[picks] - 0.5 * share[by_index][picks]
    return u, ids[by_index][picks], np.log(share[by_index][picks])


def draw(rv, rows, u, T=None, k=None, p=None, mp=None):
    n = len(u)
    full = lambda v, make: None if v is None else make([v] * n)  # noqa: E731
    return rv.sample(rows, f32(u), full(T, f32), full(k, i32), full(p, f32), full(mp, f32))


@pytest.mark.parametrize("n", [1, 2, 31, 1000, 4097, 49999, 151936])
@pytest.mark.parametrize("T,k,p,mp", [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.3, 0, 0.9, 0.0), (0.5, 0, 1.0, 0.03),
                                      (2.0, 300, 0.97, 0.001), (1.0, 1, 1.0, 0.0), (1.0, 7, 0.0, 0.0)])
def test_sample_draws_the_token_of_u(rv, n, T, k, p, mp):
    rng = np.random.default_rng(n + k)
    l = (2.5 * rng.standard_normal(n)).astype(np.float32)
    # A cutoff of top-p or min-p that lies within rounding of a token would
    # make the kept set ambiguous: p and mp go to the middle of a step.
    ids, share = kept_64(l, T, k, 1.0, 0.0)
    if 0 < p < 1:
        edges = np.cumsum(share)
        at = int(np.searchsorted(edges, p))
        p = float(np.float32(edges[at] - 0.5 * share[at]))
    if mp > 0:
        at = max(0, int((share / share[0] >= mp).sum()) - 1)
        nxt = share[at + 1] / share[0] if at + 1 < len(share) else 0.0
        mp = float(np.float32(0.5 * (share[at] / share[0] + nxt)))
    u, token, logp = middle_u(l, T, k, p, mp, rng, 16)
    rows = torch.from_numpy(l).cuda().expand(16, n).contiguous()
    got, lp = draw(rv, rows, u, T, k, p, mp)
    assert got.tolist() == token.tolist()
    # z is off by two roundings (2^-23 |z|), the sum by its weights' (2^-22) and the logarithm's
    assert np.allclose(lp.double().cpu().numpy(), logp, rtol=2.0 ** -20, atol=2.0 ** -20)


def test_sample_rows_of_their_own_parameters_and_strides(rv):
    rng = np.random.default_rng(5)
    n, rows = 5003, 200
    wide = torch.from_numpy((2 * rng.standard_normal((rows, n + 13))).astype(np.float32)).cuda()
    l = wide[:, 5:5 + n]
    T = rng.uniform(0.3, 2.0, rows).astype(np.float32)
    k = rng.integers(0, 100, rows).astype(np.int32)
    want, u, lps = [], [], []
    for r in range(rows):
        uu, token, lp = middle_u(l[r].cpu().numpy(), float(T[r]), int(k[r]), 1.0, 0.0, rng, 1)
        want.append(int(token[0])), u.append(uu[0]), lps.append(lp[0])
    got, lp = rv.sample(l, f32(u), torch.from_numpy(T).cuda(), torch.from_numpy(k).cuda())
    assert got.tolist() == want
    assert np.allclose(lp.double().cpu().numpy(), lps, rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.parametrize("n", [5, 700, 40000])
def test_sample_ties_go_to_the_lowest_index(rv, n):
    """All logits equal: k tokens of equal weight are the first k indices; of
    two values, a cutoff inside the lower one keeps its first indices; exact
    (weights are powers of two)."""
    for k in (1, 2, 3, n // 2 + 1, n - 1):
        u = (np.arange(min(k, 64)) * (k // min(k, 64)) + 0.5) / k
        rows = torch.full((len(u), n), -3.25, device="cuda")
        got, lp = draw(rv, rows, u, 1.0, k)
        assert got.tolist() == [int(x * k) for x in u]
        assert np.allclose(lp.cpu().numpy(), -math.log(k), rtol=1e-6, atol=1e-6)
    # index 3 has the largest logit, all others are alike: top-k keeps 3 and 0..k-2
    rows = torch.zeros(4, n, device="cuda")
    rows[:, 3] = 1.0
    kk = min(n - 1, 4)
    ids = sorted([3] + list(range(kk - 1)))
    share = np.array([math.e if i == 3 else 1.0 for i in ids])
    edges = np.cumsum(share / share.sum())
    got, _ = draw(rv, rows, (edges - 0.5 * share / share.sum())[:4], 1.0, kk)
    assert got.tolist() == ids[:4]
    # top-p of equal weights: p = (m - 1/2) / n keeps the first m
    for m in (1, 2, n // 2, n - 1):
        rows = torch.zeros(2, n, device="cuda")
        got, _ = draw(rv, rows, [0.0, 1.0 - 2.0 ** -24], 1.0, 0, float(np.float32((m - 0.5) / n)))
        assert got.tolist() == [0, m - 1]


def test_sample_edges(rv):
    inf, nan = math.inf, math.nan
    # nothing to draw from; NaN counts as -infinity; one candidate; +infinity outweighs the rest
    rows = f32([[-inf] * 4, [nan, -inf, nan, nan], [-inf, -inf, 2.0, nan], [1.0, inf, 3.0, inf], [nan, 5.0, 5.0, -inf]])
    got, lp = draw(rv, rows, [0.3, 0.3, 0.999, 0.75, 0.75], 1.0)
    assert got.tolist() == [0, 0, 2, 3, 2]
    assert lp.tolist()[:3] == [-inf, -inf, 0.0] and abs(lp[3].item() + math.log(2)) < 1e-6
    # greedy at temperature 0, the first of equal largest (-0 and 0 are equal)
    rows = f32([[1.0, 3.0, 3.0, 2.0], [-0.0, 0.0, -1.0, -2.0], [-inf] * 4])
    got, lp = draw(rv, rows, [0.9, 0.9, 0.9], 0.0, 3, 0.9, 0.1)
    assert got.tolist() == [1, 0, 0] and lp.tolist() == [0.0, 0.0, -inf]
    # u at its ends and outside [0, 1)
    rows = f32([[0.0, 0.0, -inf, 0.0]] * 4)
    got, _ = draw(rv, rows, [0.0, 1.0 - 2.0 ** -24, 1.0, -1.0])
    assert got.tolist() == [0, 3, 3, 0]
    # min_p above 1 keeps the largest alone; a tiny temperature too
    rows = f32([[0.0, 2.0, 1.9]] * 2)
    assert draw(rv, rows, [0.0, 0.99], 1.0, 0, 1.0, 1.5)[0].tolist() == [1, 1]
    assert draw(rv, rows, [0.0, 0.99], 1e-30)[0].tolist() == [1, 1]
    assert draw(rv, rows, [0.0, 0.99], inf)[0].tolist() == [0, 2]


def test_sample_agrees_with_argmax_and_repeats(rv):
    l = torch.randn(50, 151936, device="cuda", generator=gen(41))
    got, _ = draw(rv, l, [0.5] * 50, 0.0)
    assert got.tolist() == l.argmax(1).tolist()
    u = torch.rand(50, device="cuda", generator=gen(42)).tolist()
    a = draw(rv, l, u, 1.1, 40000, 0.95, 1e-6)
    for _ in range(3):
        b = draw(rv, l, u, 1.1, 40000, 0.95, 1e-6)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_sample_frequencies(rv):
    """20,000 draws of 8 tokens: each count within 5 standard deviations."""
    l = np.array([0.0, 1.0, -1.0, 2.0, 0.5, -2.0, 1.5, -3.0], np.float32)
    rows = torch.from_numpy(l).cuda().expand(20000, 8).contiguous()
    got, _ = rv.sample(rows, torch.rand(20000, device="cuda", generator=gen(43)))
    share = np.exp(l.astype(np.float64)) / np.exp(l.astype(np.float64)).sum()
    count = np.bincount(got.cpu().numpy(), minlength=8)
    assert (np.abs(count - 20000 * share) < 5 * np.sqrt(20000 * share * (1 - share))).all()
