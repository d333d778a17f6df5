"""Refusals of the operators that decode a batch of continuations of one
prompt: bad geometry and arguments are found before any CUDA call."""
import ctypes

import pytest

F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def rv():
    import ramvamp_b200

    return ramvamp_b200


@pytest.fixture()
def name(rv):
    return lambda code: rv.lib().rv_status_name(code).decode()


def cache(rv, format=0, n_seqs=2, heads=4, dim=128, capacity=64, k=0x1000, v=0x1000, ks=0x1000, vs=0x1000):
    from ramvamp_b200 import _lib

    return _lib.KvCacheC(format, n_seqs, heads, dim, capacity, k, v, ks, vs)


def append(rv, c, dtype=F32, k=0x1000, v=0x1000, seq=2048, token=512, n=2, lens=None, position=0):
    return rv.lib().rv_kv_append(None if c is None else ctypes.addressof(c), dtype, k, v, seq, token, n, lens, position, None)


def test_kv_refusals(rv, name):
    assert name(append(rv, None)) == "InvalidArgument"
    for bad, kind in ((dict(format=2), "UnsupportedFormat"), (dict(n_seqs=0), "Empty"), (dict(heads=0), "Empty"),
                      (dict(dim=0), "InvalidHeadDim"), (dict(dim=129), "InvalidHeadDim"), (dict(dim=100), "Unimplemented"),
                      (dict(dim=264), "Unimplemented"), (dict(capacity=1 << 31), "Unimplemented"),
                      (dict(n_seqs=65536), "Unimplemented"), (dict(capacity=1), "CapacityExceeded"),
                      (dict(k=None), "InvalidArgument"), (dict(v=0x1008), "InvalidArgument"),
                      (dict(format=1, ks=None), "InvalidArgument"), (dict(format=1, vs=0x1002), "InvalidArgument")):
        assert name(append(rv, cache(rv, **bad))) == kind, bad
    c = cache(rv)
    for bad, kind in ((dict(dtype=3), "UnsupportedFormat"), (dict(dtype=-1), "UnsupportedFormat"),
                      (dict(position=63), "CapacityExceeded"), (dict(position=2 ** 63), "CapacityExceeded"),
                      (dict(n=65), "CapacityExceeded"), (dict(k=None), "InvalidArgument"), (dict(v=0x1002), "InvalidArgument"),
                      (dict(lens=0x1001), "InvalidArgument"), (dict(token=511), "LengthMismatch")):
        assert name(append(rv, c, **bad)) == kind, bad
    assert append(rv, c, n=0, k=None, v=None) == 0
    read = rv.lib().rv_kv_read
    ref = ctypes.addressof(c)
    assert name(read(None, F32, 2, None, 0, 0x1000, 0x1000, None)) == "InvalidArgument"
    assert name(read(ref, 9, 2, None, 0, 0x1000, 0x1000, None)) == "UnsupportedFormat"
    assert name(read(ref, F16, 65, None, 0, 0x1000, 0x1000, None)) == "CapacityExceeded"
    assert name(read(ref, F16, 2, None, 0, None, 0x1000, None)) == "InvalidArgument"
    assert read(ref, F16, 0, None, 0, None, None, None) == 0


def attend(rv, prefix, prefix_len, suffix, lens=0x1000, dtype=F32, q=0x1000, n_q=1, heads=32, out=0x1000, scratch=0x1000,
           scratch_len=1 << 40):
    ref = lambda c: None if c is None else ctypes.addressof(c)  # noqa: E731
    return rv.lib().rv_prefix_attention(ref(prefix), prefix_len, ref(suffix), lens, dtype, q, 4096, 4096, n_q, heads,
                                        ctypes.c_float(0.1), out, scratch, scratch_len, None)


def test_prefix_attention_refusals(rv, name):
    pre, suf = cache(rv, n_seqs=1), cache(rv)
    assert name(attend(rv, pre, 10, None)) == "InvalidArgument"
    assert name(attend(rv, None, 10, suf)) == "InvalidArgument"
    assert name(attend(rv, cache(rv, n_seqs=1, format=1), 10, suf)) == "UnsupportedFormat"
    assert name(attend(rv, cache(rv, n_seqs=2), 10, suf)) == "LengthMismatch"
    assert name(attend(rv, cache(rv, n_seqs=1, heads=2), 10, suf)) == "LengthMismatch"
    assert name(attend(rv, cache(rv, n_seqs=1, dim=64), 10, suf)) == "LengthMismatch"
    assert name(attend(rv, pre, 65, suf)) == "CapacityExceeded"
    assert name(attend(rv, cache(rv, n_seqs=1, k=None), 10, suf)) == "InvalidArgument"
    for bad, kind in ((dict(dtype=BF16), "UnsupportedFormat"), (dict(heads=0), "Empty"), (dict(heads=30), "LengthMismatch"),
                      (dict(n_q=65536), "Unimplemented"), (dict(q=None), "InvalidArgument"), (dict(q=0x1002), "InvalidArgument"),
                      (dict(out=None), "InvalidArgument"), (dict(lens=None), "InvalidArgument"),
                      (dict(lens=0x1002), "InvalidArgument"), (dict(scratch=None), "InvalidArgument"),
                      (dict(scratch=0x1008), "InvalidArgument"), (dict(scratch_len=0), "LengthMismatch")):
        assert name(attend(rv, pre, 10, suf, **bad)) == kind, bad
    assert attend(rv, pre, 10, suf, n_q=0) == 0
    size = rv.lib().rv_prefix_attention_scratch
    n = ctypes.c_size_t()
    assert name(size(1, 1, 32, 4, 128, None)) == "InvalidArgument"
    assert name(size(1, 1, 32, 0, 128, ctypes.byref(n))) == "Empty"
    assert name(size(1, 1, 32, 5, 128, ctypes.byref(n))) == "LengthMismatch"


def test_sample_refusals(rv, name):
    def call(logits=0x1000, stride=100, rows=2, n=100, u=0x1000, t=None, k=None, p=None, mp=None, tokens=0x1000, lp=None):
        return rv.lib().rv_sample(logits, stride, rows, n, u, t, k, p, mp, tokens, lp, None)

    for bad, kind in ((dict(n=0), "Empty"), (dict(n=720897, stride=1 << 22), "Unimplemented"), (dict(rows=1 << 31), "Unimplemented"),
                      (dict(stride=99), "LengthMismatch"), (dict(logits=None), "InvalidArgument"), (dict(u=None), "InvalidArgument"),
                      (dict(tokens=None), "InvalidArgument"), (dict(t=0x1001), "InvalidArgument"), (dict(k=0x1002), "InvalidArgument"),
                      (dict(lp=0x1003), "InvalidArgument")):
        assert name(call(**bad)) == kind, bad
    assert call(rows=0) == 0


def test_python_checks(rv):
    torch = pytest.importorskip("torch")
    with pytest.raises(rv.KernelError) as e:
        rv.KvCache.of(torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 3, 8))
    assert e.value.kind == "UnsupportedFormat"
    k = torch.zeros(1, 2, 3, 8, dtype=torch.int8)
    for scales in ((None, None), (torch.zeros(1, 2, 3), torch.zeros(1, 2, 4)), (torch.zeros(1, 2, 3).double(), torch.zeros(1, 2, 3))):
        with pytest.raises(rv.KernelError) as e:
            rv.KvCache.of(k, k, *scales)
        assert e.value.kind == "LengthMismatch"
    c = rv.KvCache.of(k, k, torch.zeros(1, 2, 3), torch.zeros(1, 2, 3))
    with pytest.raises(rv.KernelError):
        rv.KvCache.of(k.half(), k.half(), torch.zeros(1, 2, 3), None)
    x = torch.zeros(1, 1, 3, 8)
    for bad in (torch.zeros(1, 1, 3, 16), torch.zeros(2, 1, 3, 8), torch.zeros(1, 1, 8, 3).transpose(2, 3)):
        with pytest.raises(rv.KernelError):
            rv.kv_append(c, bad, bad)
    with pytest.raises(rv.KernelError):
        rv.kv_append(c, x, x.half())
    with pytest.raises(rv.KernelError):
        rv.kv_append(c, x, x, lens=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(rv.KernelError):
        rv.prefix_attention(torch.zeros(1, 1, 6, 16), None, 0, c, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(rv.KernelError):
        rv.prefix_attention(torch.zeros(1, 1, 6, 8), None, 0, c, torch.zeros(1, dtype=torch.int32), out=torch.zeros(1, 1, 6, 8).half())
    for logits in (torch.zeros(4), torch.zeros(2, 4).half(), torch.zeros(4, 2).t()):
        with pytest.raises(rv.KernelError):
            rv.sample(logits, torch.zeros(2))
    with pytest.raises(rv.KernelError):
        rv.sample(torch.zeros(2, 4), torch.zeros(3))
    with pytest.raises(rv.KernelError):
        rv.sample(torch.zeros(2, 4), torch.zeros(2), top_k=torch.zeros(2))


def test_host_tensors_are_refused(rv):
    """Right in shape and type, but in host memory: refused before a pointer reaches a kernel."""
    torch = pytest.importorskip("torch")
    z = torch.zeros
    c = rv.KvCache.of(z(1, 2, 3, 8).half(), z(1, 2, 3, 8).half())
    lens = z(1, dtype=torch.int32)
    for call in (lambda: rv.kv_append(c, z(1, 1, 3, 8), z(1, 1, 3, 8), lens=lens), lambda: rv.kv_read(c, 1),
                 lambda: rv.prefix_attention(z(1, 1, 6, 8), None, 0, c, lens), lambda: rv.sample(z(2, 4), z(2)),
                 lambda: rv.prefix_attention(z(1, 1, 6, 8), None, 0, c, None)):
        with pytest.raises(rv.KernelError) as e:
            call()
        assert e.value.kind == "InvalidArgument"
    # a cache on a GPU and host tensors beside it (the check comes before any pointer is used)
    c._index = 0
    for call in (lambda: rv.kv_append(c, z(1, 1, 3, 8), z(1, 1, 3, 8)), lambda: rv.kv_read(c, 1, lens=lens),
                 lambda: rv.prefix_attention(z(1, 1, 6, 8), None, 0, c, lens)):
        with pytest.raises(rv.KernelError) as e:
            call()
        assert e.value.kind == "InvalidArgument"
