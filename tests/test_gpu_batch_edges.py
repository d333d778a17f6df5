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
