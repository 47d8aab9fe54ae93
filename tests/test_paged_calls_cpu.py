"""Paged cache without a GPU: calls whose outputs share memory with what they read, and pages for all sequences or none."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

# one array after the other: a cache of 2 layers and 3 sequences, 5 rows a sequence
PLACES = {name: (i + 1) << 20 for i, name in enumerate(
    ["keys", "values", "table", "lengths", "tokens", "parents", "choices", "counts", "accepted", "taken", "status", "q", "k", "v", "inv_freq",
     "depths", "visible", "out", "scratch"])}


def cache():
    from kotensor_b200 import _lib
    at = {n: PLACES[n] for n in ("keys", "values", "table", "lengths")}
    return _lib.KtPagedCache(**at, layers=2, batch=3, kv_heads=2, head_dim=64, pages=5, page=16, width=4, table_stride=6, dtype=_lib.KT_BF16)


def refused(lib, status):
    return status == 1 and "overlap" in lib.kt_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(accepted="choices"), dict(accepted="tokens"), dict(accepted="parents"), dict(accepted=("choices", 56)), dict(accepted=("choices", -56)),
    dict(accepted="counts"), dict(accepted=("lengths", 8)), dict(accepted="table"), dict(accepted=("table", 5 * 6 * 4 - 60 - 8)), dict(taken="counts"), dict(taken="lengths"),
    dict(taken=("tokens", 59)), dict(taken=("parents", -8)), dict(taken=("table", 24 * 2 + 12)), dict(taken="accepted"), dict(taken=("accepted", 56)),
    dict(status="lengths"), dict(status=("accepted", 4)), dict(status=("taken", 8)), dict(status=("choices", 56)), dict(status="counts"),
])
def test_accepted_paths_over_what_is_read(kt, change):
    lib = kt.load_library()
    at = dict(PLACES)
    for name, place in change.items():
        at[name] = PLACES[place] if isinstance(place, str) else PLACES[place[0]] + place[1]
    assert refused(lib, lib.kt_paged_accept(ctypes.c_void_p(4096), ctypes.byref(cache()), at["tokens"], at["parents"], at["choices"], 5, at["counts"],
                                            at["accepted"], at["taken"], at["status"], None))


@pytest.mark.parametrize("change", [
    dict(out="q"), dict(out=("q", 104)), dict(out="k"), dict(out=("v", 14 * 1024 + 504)), dict(out=("v", -7672)), dict(out="inv_freq"), dict(out=("counts", 8)),
    dict(out=("depths", 56)), dict(out="lengths"), dict(out=("table", 64 - 8)), dict(status="counts"), dict(status=("q", 14 * 1024 + 1020)),
    dict(status=("depths", 56)), dict(status=("out", 7676)), dict(status=("table", 12)), dict(status="lengths"), dict(status=("inv_freq", 124)),
])
def test_appended_queries_over_what_is_read(kt, change):
    """15 rows of 4 + 2 + 2 heads of 64; rows of q, k and v lie 1024 bytes apart."""
    lib = kt.load_library()
    at = dict(PLACES)
    for name, place in change.items():
        at[name] = PLACES[place] if isinstance(place, str) else PLACES[place[0]] + place[1]
    assert refused(lib, lib.kt_paged_append(ctypes.c_void_p(4096), ctypes.byref(cache()), 0, at["q"], at["k"], at["v"], 256, 256, 256, 4,
                                            at["inv_freq"], 5, at["counts"], at["depths"], at["out"], at["status"], None))


@pytest.mark.parametrize("change,stride,dtype", [
    (dict(out="q"), 264, 1), (dict(out="q"), 256, 0), (dict(out=("q", 2)), 256, 1), (dict(out=("q", -7678)), 256, 1),
    (dict(out=("q", 14 * 1024 + 510)), 512, 1), (dict(out=("counts", 8)), 256, 1), (dict(out="visible"), 256, 1), (dict(out=("visible", 56)), 256, 1),
    (dict(out=("lengths", 8)), 256, 1), (dict(out=("table", 60)), 256, 0),
])
def test_attention_over_what_it_reads(kt, change, stride, dtype):
    lib = kt.load_library()
    at = dict(PLACES)
    for name, place in change.items():
        at[name] = PLACES[place] if isinstance(place, str) else PLACES[place[0]] + place[1]
    assert refused(lib, lib.kt_paged_attention(ctypes.c_void_p(4096), ctypes.byref(cache()), 0, at["q"], stride, at["out"], dtype, 5, at["counts"],
                                               at["visible"], 4, 1.0, at["scratch"], None))


def pool(batch, pages):
    """A cache's table and pool on the CPU: pages of 16 slots, 8 to a sequence."""
    from kotensor_b200.paged import PagedKVCache
    c = object.__new__(PagedKVCache)
    c.batch, c.page, c.capacity, c._first, c.device = batch, 16, 128, 0, torch.device("cpu")
    c._free, c._own = list(range(pages - 1, -1, -1)), [[] for _ in range(batch)]
    c.table, c.lengths = torch.full((batch, 8), -1, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
    return c


def test_pages_for_all_sequences_or_none():
    c = pool(3, 10)
    with pytest.raises(ValueError, match="12 pages wanted, 10 are free"):
        c.reserve(range(3), 50)
    assert c.free_pages == 10 and (c.table == -1).all()
    c.reserve([0, 0, 2], 20)  # (a sequence twice is one)
    assert c.free_pages == 6 and [len(o) for o in c._own] == [2, 0, 2]
    c.reserve(range(3), 48)
    assert c.free_pages == 1 and (c.table >= 0).sum(1).tolist() == [3, 3, 3]
    assert len(set(c.table[c.table >= 0].tolist())) == 9 and [c.table[b, :3].tolist() for b in range(3)] == c._own
    with pytest.raises(ValueError, match="3 pages wanted, 1 are free"):
        c.reserve(range(3), 49)
    with pytest.raises(ValueError, match="sequence 3 of 3"):
        c.reserve([0, 3], 64)
    with pytest.raises(ValueError, match="do not fit"):
        c.reserve(range(3), 129)
    assert c.free_pages == 1
    c.reserve(torch.tensor(1), 64)
    c.release(0)
    assert c.free_pages == 3


def test_pages_that_could_not_be_written_down_stay_free(monkeypatch):
    c = pool(2, 6)
    monkeypatch.setattr(torch, "tensor", lambda *a, **k: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        c.reserve(0, 40)
    assert c.free_pages == 6 and c._own == [[], []]
