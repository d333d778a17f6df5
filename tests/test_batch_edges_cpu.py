"""What the Python entry points of the batched-continuation operators let
through to the kernels, with the library stubbed: no GPU, no launch."""
import pytest

torch = pytest.importorskip("torch")


class Stub:
    """Stands for the loaded library: records the calls it gets."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


@pytest.fixture()
def rv():
    import ramvamp_b200

    return ramvamp_b200


@pytest.fixture()
def on_gpu(rv, monkeypatch):
    """on_gpu(tensors', current): tensors say that they are on one GPU while
    another (or the same) is current; the stub in the library's place."""

    def set_up(index, current):
        stub = Stub()
        monkeypatch.setattr(rv, "lib", lambda: stub)
        monkeypatch.setattr(torch.Tensor, "get_device", lambda self: index, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
        return stub

    return set_up


def calls(rv):
    """(name, call) of the four operators on tensors that they accept."""
    z = torch.zeros
    c = rv.KvCache.of(z(1, 2, 3, 8).half(), z(1, 2, 3, 8).half())
    lens, scratch = z(1, dtype=torch.int32), z(1 << 16, dtype=torch.uint8)
    return {
        "rv_kv_append": lambda: rv.kv_append(c, z(1, 1, 3, 8), z(1, 1, 3, 8), lens=lens),
        "rv_kv_read": lambda: rv.kv_read(c, 1, lens=lens),
        "rv_prefix_attention": lambda: rv.prefix_attention(z(1, 1, 6, 8), c, 2, c, lens, scratch=scratch),
        "rv_sample": lambda: rv.sample(z(2, 4), z(2)),
    }


@pytest.mark.parametrize("name", ["rv_kv_append", "rv_kv_read", "rv_prefix_attention", "rv_sample"])
def test_tensors_of_a_gpu_that_is_not_current_are_refused(rv, on_gpu, name):
    """The stream and the kernels are the current device's: pointers of another
    GPU must not reach them."""
    stub = on_gpu(1, current=0)
    with pytest.raises(rv.KernelError) as e:
        calls(rv)[name]()
    assert e.value.kind == "InvalidArgument" and stub.calls == []
    stub = on_gpu(1, current=1)
    calls(rv)[name]()
    assert [c[0] for c in stub.calls] == [name]


def test_the_parallel_decoder_runs_on_its_own_device(rv, monkeypatch):
    """prefill, step and generate make the decoder's device current."""
    from ramvamp_b200.model import ParallelDecoder

    seen = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            seen.append(self.index)

        def __exit__(self, *exc):
            seen.append("out")

    monkeypatch.setattr(torch.cuda, "device", Device)
    par = object.__new__(ParallelDecoder)
    par.device, par.prompt_len, par.new, par.max_new, par.max_prompt, par.n = 1, 0, 0, 4, 4, 2
    par.w = par.cfg = None
    for call, error in ((lambda: par.prefill([]), ValueError), (lambda: par.step(torch.zeros(2)), (ValueError, AttributeError)),
                        (lambda: par.generate([1], 2), AttributeError)):
        seen.clear()
        with pytest.raises(error):
            call()
        assert seen == [1, "out"]


def test_scratch_with_gaps_is_refused(rv, on_gpu):
    """A view of every other byte: as many elements as bytes are needed, but the
    kernels would write between them and past them."""
    stub = on_gpu(0, current=0)
    z = torch.zeros
    c = rv.KvCache.of(z(1, 2, 3, 8).half(), z(1, 2, 3, 8).half())
    lens, wide = z(1, dtype=torch.int32), z(1 << 16, 2, dtype=torch.uint8)
    with pytest.raises(rv.KernelError) as e:
        rv.prefix_attention(z(1, 1, 6, 8), c, 2, c, lens, scratch=wide[:, 0])
    assert e.value.kind == "LengthMismatch" and stub.calls == []
    rv.prefix_attention(z(1, 1, 6, 8), c, 2, c, lens, scratch=wide)
    assert [x[0] for x in stub.calls] == ["rv_prefix_attention"]


def test_strides_of_one_token_or_sequence_do_not_matter(rv, on_gpu):
    """k and v that differ only in the stride of a dimension of size 1 are alike;
    where it counts, different strides are still refused."""
    stub = on_gpu(0, current=0)
    z = torch.zeros(4096)

    def rows(n_seqs, n, seq, token, heads=3, head=8):
        return z.as_strided((n_seqs, n, heads, 8), (seq, token, head, 1))

    def cache(n_seqs, heads=3):
        return rv.KvCache.of(torch.zeros(n_seqs, 4, heads, 8).half(), torch.zeros(n_seqs, 4, heads, 8).half())

    rv.kv_append(cache(1), rows(1, 1, 24, 24), rows(1, 1, 7, 5))          # a sequence's only new token
    rv.kv_append(cache(4), rows(4, 1, 100, 24), rows(4, 1, 100, 100))     # one token of each
    rv.kv_append(cache(1), rows(1, 3, 72, 40), rows(1, 3, 1, 40))         # a prompt
    rv.kv_append(cache(2, 1), rows(2, 2, 64, 16, 1, 8), rows(2, 2, 64, 16, 1, 3))  # one head
    assert [(x[0], x[1][4:7]) for x in stub.calls] == [("rv_kv_append", (24, 24, 1)), ("rv_kv_append", (100, 24, 1)),
                                                       ("rv_kv_append", (120, 40, 3)), ("rv_kv_append", (64, 16, 2))]
    for n_seqs, k, v in ((4, rows(4, 1, 100, 24), rows(4, 1, 101, 24)), (1, rows(1, 3, 72, 40), rows(1, 3, 72, 41)),
                         (1, rows(1, 3, 72, 40), rows(1, 2, 72, 40)), (1, rows(1, 1, 24, 24), rows(1, 1, 24, 24, 3, 9))):
        with pytest.raises(rv.KernelError) as e:
            rv.kv_append(cache(n_seqs), k, v)
        assert e.value.kind == "LengthMismatch"
    assert len(stub.calls) == 4


def test_sample_takes_a_row_stride_of_zero(rv):
    """The checks go on to the null pointer behind the stride's."""
    name = lambda stride: rv.lib().rv_status_name(  # noqa: E731
        rv.lib().rv_sample(None, stride, 2, 100, 0x1000, None, None, None, None, 0x1000, None, None)).decode()
    assert name(0) == name(100) == "InvalidArgument" and name(99) == name(1) == "LengthMismatch"
