"""kt_logits_process with lists that are empty and with single rows of any stride:
the same steps as with nothing in them (oracle/kv8_oracle.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,biases", [(1, 1000, 0), (2, 9001, 7), (3, 151936, 0)])
def test_an_empty_history_penalizes_nothing(kt, rows, vocab, biases):
    """tokens [rows, 0]: the first token of a text without a prompt."""
    from test_logits_gpu import case, check, run
    a = case(rows, vocab, None, biases, True, seed=vocab)
    a["tokens"] = np.zeros((rows, 0), np.int32)
    a["lengths"] = np.zeros(rows, np.int32)
    for name in ("repetition", "frequency", "presence"):
        a[name] = np.full(rows, 2.0, np.float32)
    out, token, _ = run(kt, a)
    check(a, out, token)
    a["lengths"][:] = 5  # at most the width counts
    again, second, _ = run(kt, a)
    assert torch.equal(out, again) and torch.equal(token, second)


def test_an_empty_history_at_the_c_entry(kt):
    """No tokens at all is refused where penalties are given, unless the list's width is 0."""
    from kotensor_b200 import _lib
    import ctypes
    lib, h = _lib.load(), kt.Context.get().handle
    x, one = torch.randn(1, 64, device="cuda"), torch.full((1,), 2.0, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    a = _lib.KtLogitsArgs()
    a.logits, a.out, a.logits_stride, a.out_stride, a.rows, a.vocab = x.data_ptr(), out.data_ptr(), 64, 64, 1, 64
    a.repetition, a.lengths = one.data_ptr(), n.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.kt_logits_process(h, ctypes.byref(a), stream) == 0
    assert torch.equal(out, x)
    a.token_width = 3
    assert lib.kt_logits_process(h, ctypes.byref(a), stream) == 1
    a.token_width, a.lengths = 0, None
    assert lib.kt_logits_process(h, ctypes.byref(a), stream) == 1


def test_one_row_of_any_stride(kt):
    """The stride between rows means nothing where there is one row: a column seen as a row."""
    from test_logits_gpu import case, check
    from kotensor_b200.logits import LogitsProcessor
    a = case(1, 5000, 20, 3, True, seed=1)
    dev = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    for name in ("logits", "tokens", "bias_ids", "allowed"):
        dev[name] = dev[name].reshape(-1, 1).t()
        assert dev[name].stride() == (1, 1)
    out = torch.empty(5000, 1, device="cuda").t()
    token = LogitsProcessor(1, 5000)(out=out, **dev)
    check(a, out, token)
