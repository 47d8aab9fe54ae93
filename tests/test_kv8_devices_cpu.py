"""KVCache8 and LogitsProcessor refuse tensors of another GPU than their own before
anything is launched: stand-ins for tensors and for the library, no GPU."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


class Tensor:
    """What the checks ask of a tensor."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.number = tuple(shape), dtype, device
        self.is_cuda = device >= 0

    @property
    def device(self):
        return torch.device("cuda", self.number) if self.is_cuda else torch.device("cpu")

    def get_device(self):
        return self.number

    def stride(self, i=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096

    def new_empty(self, shape):
        return Tensor(shape, self.dtype, self.number)


@pytest.fixture
def calls(monkeypatch):
    """A cache and a processor of GPU 1 whose library records its calls."""
    from kotensor_b200 import kv8, logits
    made = []

    def entry(*args):
        made.append(args)
        return 0

    for module in (kv8, logits):
        monkeypatch.setattr(module, "raw_stream", lambda device: 0)
    c = object.__new__(kv8.KVCache8)
    c.layers, c.batch, c.kv_heads, c.head_dim, c.capacity, c.block = 1, 2, 2, 16, 64, 16
    c.ctx = SimpleNamespace(handle=None, device=1)
    c.device = torch.device("cuda", 1)
    c.weights, c._scale, c._status = None, 0.25, 0
    c._layer = [(None, None)]
    c._store = c._attention = entry
    c._lib = SimpleNamespace(kt_kv8_advance=entry)
    c.lengths = Tensor([2], torch.int32, 1)
    c._scratch_of = lambda rows, heads: 4096
    p = object.__new__(logits.LogitsProcessor)
    p.rows, p.vocab, p.ctx = 2, 64, SimpleNamespace(handle=None, device=1)
    p.next_token = Tensor([2], torch.int32, 1)
    p._process, p._scratch_ptr = entry, 4096
    from kotensor_b200 import _lib
    import ctypes
    p._args = _lib.KtLogitsArgs()
    p._args_ref = ctypes.byref(p._args)
    return c, p, made


def f32(*shape, on=1):
    return Tensor(shape, torch.float32, on)


def i32(*shape, on=1):
    return Tensor(shape, torch.int32, on)


@pytest.mark.parametrize("other", [0, 2, -1])
def test_the_cache_refuses_tensors_of_another_device(calls, other):
    c, _, made = calls
    c.store(0, f32(2, 32), f32(2, 32), counts=i32(2))
    c.attend(0, f32(2, 64), 4, out=f32(2, 64), counts=i32(2))
    c.advance(1, counts=i32(2))
    assert len(made) == 3
    for bad in (lambda: c.store(0, f32(2, 32, on=other), f32(2, 32)), lambda: c.store(0, f32(2, 32), f32(2, 32, on=other)),
                lambda: c.store(0, f32(2, 32), f32(2, 32), counts=i32(2, on=other)),
                lambda: c.attend(0, f32(2, 64, on=other), 4), lambda: c.attend(0, f32(2, 64), 4, out=f32(2, 64, on=other)),
                lambda: c.attend(0, f32(2, 64), 4, counts=i32(2, on=other)),
                lambda: c.advance(1, counts=i32(2, on=other))):
        with pytest.raises(ValueError):
            bad()
    assert len(made) == 3


@pytest.mark.parametrize("other", [0, 2, -1])
def test_the_processor_refuses_tensors_of_another_device(calls, other):
    _, p, made = calls
    good = dict(logits=f32(2, 64), out=f32(2, 64), tokens=i32(2, 5), lengths=i32(2), prompt_lengths=i32(2), repetition=f32(2),
                frequency=f32(2), presence=f32(2), bias_ids=i32(2, 3), bias_values=f32(2, 3), bias_counts=i32(2),
                allowed=i32(2, 2), next_token=i32(2))
    p(**good)
    assert len(made) == 1
    for name, x in good.items():
        with pytest.raises(ValueError):
            p(**{**good, name: Tensor(x.shape, x.dtype, other)})
    assert len(made) == 1
