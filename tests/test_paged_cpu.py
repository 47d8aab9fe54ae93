"""Paged cache without a GPU: what the C entries and the Python class refuse before any
launch, and the masks of drafted trees."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def good(**change):
    from kotensor_b200 import _lib
    fields = dict(keys=4096, values=4096, table=4096, lengths=4096, layers=2, batch=3, kv_heads=2, head_dim=64, pages=5, page=16,
                  width=4, table_stride=4, dtype=_lib.KT_BF16)
    return _lib.KtPagedCache(**{**fields, **change})


BAD_CACHES = [
    (dict(keys=None), "NULL argument"), (dict(table=None), "NULL argument"), (dict(lengths=None), "NULL argument"),
    (dict(keys=4104), "16-byte aligned"), (dict(head_dim=48), "head_dim"), (dict(head_dim=72), "head_dim"), (dict(head_dim=144), "head_dim"),
    (dict(page=48), "page must be"), (dict(page=256), "page must be"), (dict(pages=0), "must be positive"), (dict(width=0), "must be positive"),
    (dict(batch=0), "batch"), (dict(batch=40000), "batch"), (dict(kv_heads=0), "kv_heads"), (dict(dtype=0), "dtype"), (dict(dtype=3), "dtype"),
    (dict(table_stride=3), "table"), (dict(width=1 << 27, table_stride=1 << 27), "2\\^30"), (dict(pages=1 << 28), "too many rows"),
]


def calls(lib, ctx, cache, layer=0, rows=1, heads=4, q=4096, q_stride=256, k_stride=128, out_dtype=1, scratch=4096, visible=None,
          q_out=4096):
    ref = ctypes.byref(cache)
    return {
        "append": lambda: lib.kt_paged_append(ctx, ref, layer, q, 4096, 4096, q_stride, k_stride, 128, heads, 4096, rows, None, None, q_out,
                                              None, None),
        "attend": lambda: lib.kt_paged_attention(ctx, ref, layer, q, q_stride, 4096, out_dtype, rows, None, visible, heads, 1.0,
                                                 scratch, None),
        "accept": lambda: lib.kt_paged_accept(ctx, ref, 4096, 4096, 4096, rows, None, 4096, 4096, None, None),
    }


@pytest.mark.parametrize("change,message", BAD_CACHES)
def test_caches_that_are_refused(kt, change, message):
    import re
    lib = kt.load_library()
    ctx = ctypes.c_void_p(4096)  # the checks come before its use
    for name, call in calls(lib, ctx, good(**change)).items():
        assert call() == 1, name
        assert re.search(message, lib.kt_last_error().decode()), (name, lib.kt_last_error())


@pytest.mark.parametrize("name,change,message", [
    ("append", dict(layer=2), "layer"), ("append", dict(layer=-1), "layer"), ("append", dict(rows=-1), "Negative"),
    ("append", dict(k_stride=127), "shorter"), ("append", dict(q_stride=255), "shorter"), ("append", dict(heads=0), "heads"),
    ("append", dict(q=None), "heads"), ("append", dict(q_out=None), "NULL"), ("append", dict(q_out=4100), "8-byte"),
    ("append", dict(rows=1 << 30), "too many rows"),
    ("attend", dict(layer=2), "layer"), ("attend", dict(rows=-1), "Negative"), ("attend", dict(q=None), "NULL"), ("attend", dict(heads=3), "multiple"),
    ("attend", dict(heads=0), "multiple"), ("attend", dict(q_stride=100), "shorter"), ("attend", dict(out_dtype=2), "out_dtype"),
    ("attend", dict(scratch=4100), "scratch"), ("attend", dict(scratch=None), "NULL"), ("attend", dict(rows=1025, visible=4096), "1024"),
    ("attend", dict(rows=1 << 29), "too many rows"), ("attend", dict(rows=1 << 28, heads=12, q_stride=768), "too many rows"),
    ("accept", dict(rows=0), "1..1024"), ("accept", dict(rows=1025), "1..1024"),
])
def test_calls_that_are_refused(kt, name, change, message):
    lib = kt.load_library()
    assert calls(lib, ctypes.c_void_p(4096), good(), **change)[name]() == 1
    assert message in lib.kt_last_error().decode()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])  # (3e38 * log2(e) is past fp32)
def test_scales_that_are_refused(kt, scale):
    lib = kt.load_library()
    assert lib.kt_paged_attention(ctypes.c_void_p(4096), ctypes.byref(good()), 0, 4096, 256, 4096, 1, 1, None, None, 4, scale, 4096, None) == 1
    assert "scale" in lib.kt_last_error().decode()


def test_more_heads_than_a_launch_counts(kt):
    lib = kt.load_library()
    assert calls(lib, ctypes.c_void_p(4096), good(), heads=65536, q_stride=1 << 22)["attend"]() == 1
    assert "65535" in lib.kt_last_error().decode()


def test_no_context_and_no_rows(kt):
    lib = kt.load_library()
    for call in calls(lib, None, good()).values():
        assert call() == 1
    made = calls(lib, ctypes.c_void_p(4096), good(), rows=0)
    assert made["append"]() == 0 and made["attend"]() == 0
    assert lib.kt_paged_scratch_bytes(None) == 0


class Tensor:
    """What the checks ask of a tensor."""

    def __init__(self, shape, dtype, device=1, strides=None):
        self.shape, self.dtype, self.number, self.strides = torch.Size(shape), dtype, device, strides

    device = property(lambda self: torch.device("cuda", self.number))

    def get_device(self):
        return self.number

    def stride(self):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return self.strides or tuple(s)

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return self.strides is None

    def data_ptr(self):
        return 4096


@pytest.fixture
def cache(monkeypatch):
    """A cache of GPU 1 whose library records its calls."""
    from kotensor_b200 import paged
    monkeypatch.setattr(paged, "raw_stream", lambda device: 0)
    c = object.__new__(paged.PagedKVCache)
    c.layers, c.batch, c.kv_heads, c.head_dim, c.capacity, c.dtype = 1, 2, 2, 64, 64, torch.bfloat16
    c.ctx, c.device = SimpleNamespace(handle=None, device=1), torch.device("cuda", 1)
    c._types = {torch.bfloat16: 1, torch.float32: 0}
    c._ref, c._status, c._scratch, c._scale, c.made = None, 0, 0, 0.125, []
    c._append = c._attention = c._accept = lambda *args: c.made.append(args) or 0
    c._lib = SimpleNamespace(kt_kv8_advance=c._append)
    c.lengths, c._results = Tensor([2], torch.int32), {}
    return c


def test_arguments_that_the_class_refuses(cache):
    f32, b16, i32 = torch.float32, torch.bfloat16, torch.int32
    kv, freq, q16 = Tensor([6, 128], f32), Tensor([32], f32), Tensor([6, 256], b16)
    out, ints = Tensor([6, 256], b16), Tensor([2, 3], i32)
    cache.append(0, Tensor([6, 256], f32), kv, kv, freq, 3, depths=ints, out=out)
    cache.attend(0, q16, 4, 3, counts=Tensor([2], i32), visible=Tensor([2, 3, 1], i32), out=out)
    cache.accept(ints, ints, ints, accepted=ints, taken=Tensor([2], i32))
    cache.advance(3, counts=Tensor([2], i32))
    assert len(cache.made) == 4
    refused = [
        lambda: cache.append(0, Tensor([6, 256], b16), kv, kv, freq, 3, out=out),
        lambda: cache.append(0, Tensor([6, 250], f32), kv, kv, freq, 3, out=out),
        lambda: cache.append(0, None, kv, kv, freq, 3, out=out),
        lambda: cache.append(0, None, Tensor([5, 128], f32), kv, freq, 3),
        lambda: cache.append(0, None, kv, Tensor([6, 128], f32, device=0), freq, 3),
        lambda: cache.append(0, None, kv, Tensor([6, 128], f32, strides=(64, 1)), freq, 3),
        lambda: cache.append(0, None, kv, kv, Tensor([64], f32), 3),
        lambda: cache.append(0, None, kv, kv, freq, 3, depths=Tensor([6], i32)),
        lambda: cache.append(1, None, kv, kv, freq, 3),
        lambda: cache.append(0, None, kv, kv, freq, 3, counts=Tensor([2], torch.int64)),
        lambda: cache.append(0, Tensor([6, 256], f32), kv, kv, freq, 3, out=Tensor([6, 256], f32)),
        lambda: cache.attend(0, Tensor([6, 256], torch.float16), 4, 3, out=out),
        lambda: cache.attend(0, Tensor([6, 256], b16, device=0), 4, 3, out=out),
        lambda: cache.attend(0, Tensor([6, 256], b16, strides=(1, 6)), 4, 3, out=out),
        lambda: cache.attend(0, q16, 4, 3, out=Tensor([6, 256], torch.float16)),
        lambda: cache.attend(0, q16, 4, 3, out=Tensor([6, 256], b16, strides=(512, 1))),
        lambda: cache.attend(0, q16, 4, 3, visible=Tensor([2, 3, 2], i32), out=out),
        lambda: cache.attend(-1, q16, 4, 3, out=out),
        lambda: cache.accept(ints, Tensor([2, 4], i32), ints, accepted=ints, taken=Tensor([2], i32)),
        lambda: cache.accept(Tensor([6], i32), ints, ints, accepted=ints, taken=Tensor([2], i32)),
        lambda: cache.advance(3, counts=Tensor([3], i32)),
    ]
    for call in refused:
        with pytest.raises(ValueError):
            call()
    assert len(cache.made) == 4


def test_masks_of_drafted_trees():
    from kotensor_b200.paged import draft_tree
    depths, visible = draft_tree([-1, 0, 0, 2, 1])
    assert depths.tolist() == [0, 1, 1, 2, 2] and visible.tolist() == [[1], [3], [5], [13], [19]]
    depths, visible = draft_tree(np.arange(-1, 69)[None].repeat(2, 0))
    assert depths[1].tolist() == list(range(70)) and visible.shape == (2, 70, 3) and visible.dtype == np.int32
    assert visible[0, 31].tolist() == [-1, 0, 0] and visible[1, 69].tolist() == [-1, -1, 63]
    for bad in ([0, 0], [-1, 1], [-1, -1], [], [[[-1]]], list(range(-1, 1025))):
        with pytest.raises(ValueError):
            draft_tree(bad)


def test_constructor_checks(kt):
    from kotensor_b200.paged import PagedKVCache
    base = dict(layers=1, batch=1, kv_heads=2, head_dim=64, pages=4, max_tokens=64, page=16)
    for change in (dict(layers=0), dict(batch=0), dict(batch=40000), dict(head_dim=48), dict(head_dim=72), dict(page=24), dict(pages=0),
                   dict(dtype=torch.float32), dict(max_tokens=0), dict(max_tokens=1 << 31), dict(pages=1 << 28)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**base, **change})
