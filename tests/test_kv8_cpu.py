"""CPU tests of the 8-bit KV cache: the float64 oracle's format against PyTorch's float8, the scale
rule, and what the C ABI and the host classes refuse before they touch a device."""
import ctypes
import threading
import time

import numpy as np
import pytest
import torch


def test_oracle_e4m3_matches_torch_float8():
    from oracle.kv8 import e4m3
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    finite = codes[np.isfinite(codes)]
    assert np.array_equal(e4m3(finite), finite)  # every e4m3 value is its own nearest
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 10.0 ** rng.integers(-5, 3, 20000),
                        (np.sort(finite)[1:] + np.sort(finite)[:-1]) / 2]).astype(np.float32)  # ties among them
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(e4m3(x), want)
    assert e4m3(1e9) == 448.0 and e4m3(-np.inf) == -448.0 and np.isnan(e4m3(np.nan))


def test_oracle_scale_is_the_smallest_power_of_two():
    from oracle.kv8 import scale_of
    for amax in [0.0, 1e-38, 448.0, np.nextafter(448.0, 449), 1.0, 0.875, 1.75, 1.7500001, 3e38] + list(np.abs(np.random.default_rng(1).standard_normal(50))):
        s = scale_of(float(amax))
        assert np.frexp(s)[0] == 0.5 and s >= 2.0 ** -120
        assert amax <= 448 * s
        assert s == 2.0 ** -120 or amax > 448 * (s / 2)


def _desc(**kw):
    from jax4j_b200._lib import Kv8CacheDesc
    d = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, layers=1, pages=4, kv_heads=2, page=32, head_dim=128)
    d.update(kw)
    return ctypes.byref(Kv8CacheDesc(*d.values()))


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=96), "head_dim must be 64 or 128"), (dict(page=24), "multiple of 16"), (dict(page=0), "multiple of 16"),
    (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "must be positive"), (dict(pages=1 << 40), "2\\^31"),
    (dict(k=(1 << 20) + 8), "16-byte aligned"), (dict(v_scale=0), "aligned")])
def test_abi_refuses_bad_cache_descriptions(kw, match):
    from jax4j_b200._lib import call
    with pytest.raises(ValueError, match=match):
        call("j4b_kv8_copy_pages", _desc(**kw), 0, None, None, None, None)


def test_abi_refuses_a_null_cache_and_a_bad_layer():
    from jax4j_b200._lib import call
    with pytest.raises(ValueError, match="null cache"):
        call("j4b_kv8_copy_pages", None, 0, None, None, None, None)
    with pytest.raises(ValueError, match="layer 1 outside"):
        call("j4b_kv8_append", _desc(), 1, 0, 0, 0, 2, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None)


def test_cache_wrap_checks_shapes():
    from jax4j_b200.kv8 import Kv8Cache

    def codes(*s):
        return torch.zeros(s, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ok = (codes(1, 3, 2, 32, 64), codes(1, 3, 2, 32, 64), torch.zeros(1, 3, 2, 2), torch.zeros(1, 3, 2, 2))
    assert Kv8Cache.wrap(*ok).page == 32
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Kv8Cache.wrap(ok[0].view(torch.uint8), *ok[1:])
    with pytest.raises(ValueError, match="multiple of 16"):
        Kv8Cache.wrap(codes(1, 3, 2, 24, 64), codes(1, 3, 2, 24, 64), *ok[2:])
    with pytest.raises(ValueError, match="head_dim"):
        Kv8Cache.wrap(codes(1, 3, 2, 32, 96), codes(1, 3, 2, 32, 96), *ok[2:])
    with pytest.raises(ValueError, match="scales"):
        Kv8Cache.wrap(*ok[:2], torch.zeros(1, 3, 2, 32), ok[3])
    with pytest.raises(ValueError, match="contiguous"):
        Kv8Cache.wrap(*ok[:3], torch.zeros(1, 3, 2, 4)[..., ::2])


def test_rope_table_holds_cos_and_sin():
    from jax4j_b200.kv8 import rope_table
    t = rope_table(50, 64, 500.0).double().numpy()
    ang = np.arange(50)[:, None] * 500.0 ** (-2.0 * np.arange(32) / 64)
    assert np.abs(t[..., 0] - np.cos(ang)).max() < 1e-7 and np.abs(t[..., 1] - np.sin(ang)).max() < 1e-7


class FakeCache:
    """A cache's sizes without its device; page copies are noted."""
    def __init__(self, pages, page):
        self.pages, self.page, self.device, self.copies = pages, page, torch.device("cpu"), []

    def copy_pages(self, src, dst, tokens=None):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.copies.append((list(src), list(dst), tokens))


def _consistent(t):
    """Every page is free or counted as often as sequences name it; the device's table is the host's."""
    named = [p for pages in t.pages for p in pages if p >= 0]
    for p in range(t.cache.pages):
        assert t.refs[p] == named.count(p)
        assert (p in t._free) == (t.refs[p] == 0)
    t._upload()
    for row, pages in zip(t.table.tolist(), t.pages):
        assert row == pages + [-1] * (t.width - len(pages))


def test_page_table_extends_and_releases():
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(6, 32), 3, 100)
    assert t.width == 4
    starts, lengths, offsets = t.extend([33, 0, 1])
    assert (starts.tolist(), lengths.tolist(), offsets.tolist()) == ([0, 0, 0], [33, 0, 1], [0, 33, 33, 34])
    assert [len(p) for p in t.pages] == [2, 0, 1] and t.free_pages == 3
    _consistent(t)
    starts, lengths, _ = t.extend([31, 64, 0])  # the first fills its second page
    assert starts.tolist() == [33, 0, 1] and lengths.tolist() == [64, 64, 1] and t.free_pages == 1
    with pytest.raises(MemoryError, match="2 pages are needed and 1 are free"):
        t.extend([1, 1, 0])
    assert t.lengths == [64, 64, 1] and t.free_pages == 1
    with pytest.raises(ValueError, match="at most 128 tokens"):
        t.extend([65, 0, 0])
    with pytest.raises(ValueError, match="one count"):
        t.extend([1, 1])
    t.release(1)
    _consistent(t)
    assert t.lengths[1] == 0 and t.free_pages == 3
    with pytest.raises(ValueError, match="slot 3"):
        t.release(3)


def test_page_table_forks_share_full_pages_and_copy_the_last():
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(8, 16), 4, 64)
    t.extend([40, 0, 0, 0])
    t.fork(0, [1, 3])
    assert t.cache.copies == [([t.pages[0][2]] * 2, [t.pages[1][2], t.pages[3][2]], [8, 8])]
    assert t.pages[1][:2] == t.pages[0][:2] == t.pages[3][:2] and len({t.pages[s][2] for s in (0, 1, 3)}) == 3
    assert t.lengths == [40, 40, 0, 40] and [t.refs[p] for p in t.pages[0]] == [3, 3, 1]
    _consistent(t)
    t.release(0)
    _consistent(t)
    with pytest.raises(ValueError, match="in use"):
        t.fork(1, [3])
    with pytest.raises(ValueError, match="named twice"):
        t.fork(1, [0, 0])
    t.extend([0, 8, 0, 0])  # 48 tokens: a whole number of pages, nothing to copy
    copies = len(t.cache.copies)
    t.fork(1, [2])
    assert len(t.cache.copies) == copies and t.pages[2] == t.pages[1]
    _consistent(t)


def test_page_table_trims_a_window_and_compacts():
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(20, 16), 2, 200)
    t.extend([150, 30])
    # the next query of slot 0 is at 150 and sees 111 .. 150 and the first 20: pages 2 .. 5 are not needed
    assert t.trim(40, 20) == 4
    assert [i for i, p in enumerate(t.pages[0]) if p < 0] == [2, 3, 4, 5]
    assert t.trim(40, 20) == 0
    _consistent(t)
    before = [list(p) for p in t.pages]
    moved = t.compact()
    used = 20 - t.free_pages
    assert moved > 0 and t.cache.copies[-1][2] is None
    assert all(p < used for pages in t.pages for p in pages)
    src, dst, _ = t.cache.copies[-1]
    to = dict(zip(src, dst))
    assert [[to.get(p, p) for p in pages] for pages in before] == t.pages
    _consistent(t)
    assert t.compact() == 0
    t.release(0)
    t.extend([1, 1])
    _consistent(t)
    with pytest.raises(ValueError, match="positive window"):
        t.trim(0)


def test_decode_calls_of_two_threads_never_share_a_workspace(monkeypatch):
    """A decode call is two launches around one workspace: until it has returned, no other thread's
    call on the stream may be given the same."""
    from jax4j_b200 import kv8
    busy, clashes = [], []

    def fake(name, *args):
        if name == "j4b_kv8_decode_workspace":
            args[-1]._obj.value = 256
            return
        work = args[-3]
        if work in busy:
            clashes.append(work)
        busy.append(work)
        time.sleep(0.01)
        busy.remove(work)
    monkeypatch.setattr(kv8, "call", fake)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    monkeypatch.setattr(kv8.Kv8Cache, "_stream", lambda self: 7)
    codes = torch.zeros(1, 3, 2, 32, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    cache = kv8.Kv8Cache.wrap(codes, codes, torch.zeros(1, 3, 2, 2), torch.zeros(1, 3, 2, 2))
    q, table, lengths = torch.zeros(1, 2, 64), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    threads = [threading.Thread(target=lambda: [cache.attention_decode(q, table, lengths) for _ in range(5)]) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not clashes


def test_page_table_on_the_device_follows_every_change():
    """Read as a user reads it, right after a call: nothing else brings it up to date."""
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(20, 16), 3, 200)

    def check():
        assert t.table.tolist() == [p + [-1] * (t.width - len(p)) for p in t.pages]
    check()
    t.extend([150, 30, 0])
    check()
    at = t.table.data_ptr()
    t.fork(1, [2])
    check()
    assert t.trim(40, 20) == 4
    check()
    t.release(1)
    check()
    assert t.compact() > 0
    check()
    assert t.table.data_ptr() == at


def test_decoder_block_refuses_before_it_changes_the_sequences():
    from types import SimpleNamespace
    from jax4j_b200.decoder import DecoderBlock
    from jax4j_b200.kv8 import PageTable
    block = DecoderBlock(None, SimpleNamespace(world=1, rank=0, heads=2))
    cache = FakeCache(9, 16)
    cache.kv_heads, cache.head_dim, cache.layers = 2, 128, 2
    t = PageTable(cache, 2, 64)
    x = [SimpleNamespace(shape=(n, 256)) for n in range(8)]

    def unchanged(match, call, *args, **kw):
        before = ([list(p) for p in t.pages], list(t.lengths), t.free_pages, t.counts)
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)
        assert before == (t.pages, t.lengths, t.free_pages, t.counts)
    unchanged("must follow layer 0", block.decode_paged, x[2], t, layer=1)  # no step yet
    t.extend([3, 2])
    unchanged("window and sinks", block.decode_paged, x[2], t, window=-1)
    unchanged("window and sinks", block.prefill_paged, x[2], t, [1, 1], sinks=-1)
    unchanged("layer 2 outside", block.decode_paged, x[2], t, layer=2)
    unchanged("layer -1 outside", block.prefill_paged, x[2], t, [1, 1], layer=-1)
    unchanged("rows for 2", block.decode_paged, x[3], t)
    unchanged("must follow layer 0", block.decode_paged, x[2], t, layer=1)  # the last step was a prefill
    unchanged("must follow layer 0", block.prefill_paged, x[5], t, [2, 3], layer=1)
    t.extend([1, 1])
    t.release(0)  # its step is over
    unchanged("must follow layer 0", block.decode_paged, x[2], t, layer=1)


def test_page_table_fork_gives_its_pages_back_if_the_copy_fails():
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(8, 16), 3, 64)
    t.extend([20, 0, 0])

    def fail(*args):
        raise RuntimeError("no copy")
    copy, t.cache.copy_pages = t.cache.copy_pages, fail
    with pytest.raises(RuntimeError, match="no copy"):
        t.fork(0, [1, 2])
    _consistent(t)
    assert t.free_pages == 6 and t.lengths == [20, 0, 0]
    t.cache.copy_pages = copy
    t.fork(0, [1, 2])
    _consistent(t)


def test_page_table_rows_of_slots_without_a_token_start_nowhere():
    from jax4j_b200.kv8 import PageTable
    t = PageTable(FakeCache(8, 16), 3, 64)
    t.extend([20, 3, 0])
    starts, lengths, offsets = t.extend([1, 0, 1])
    assert (starts.tolist(), lengths.tolist(), offsets.tolist()) == ([20, 3, 0], [21, 3, 1], [0, 1, 1, 2])
    assert [r.tolist() for r in t.rows] == [[20, -1, 0], [21, 0, 1]]


def test_row_stride_of_one_row_is_its_width():
    """PyTorch calls a tensor of one row contiguous whatever that dimension's stride is."""
    from jax4j_b200.kv8 import _rows
    assert _rows(torch.zeros(6, 1, 64).transpose(0, 1), "q") == 6 * 64
    assert _rows(torch.zeros(1, 6, 64).expand(1, 6, 64), "q") == 6 * 64
    assert _rows(torch.zeros(256, 1).t(), "qkv") == 256
    assert _rows(torch.zeros(0, 6, 64), "q") == 6 * 64
    assert _rows(torch.zeros(5, 9, 64)[:, :6], "q") == 9 * 64
    assert _rows(torch.zeros(5, 9, 64)[:1, :6], "q") == 6 * 64
    with pytest.raises(ValueError, match="dense within a row"):
        _rows(torch.zeros(6, 2, 64).transpose(0, 1), "q")


def test_copy_pages_refuses_numbers_that_32_bits_do_not_hold(monkeypatch):
    """2^32 is not page 0."""
    from jax4j_b200 import kv8
    calls = []
    monkeypatch.setattr(kv8, "call", lambda name, ref, n, src, dst, tokens, stream: calls.append((list(src), list(dst), tokens and list(tokens))))
    monkeypatch.setattr(kv8.Kv8Cache, "_stream", lambda self: 7)
    codes = torch.zeros(1, 3, 2, 32, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    cache = kv8.Kv8Cache.wrap(codes, codes, torch.zeros(1, 3, 2, 2), torch.zeros(1, 3, 2, 2))
    for src, dst, tokens in (([2 ** 32], [1], None), ([0], [2 ** 32 + 1], None), ([0], [1], [2 ** 32 + 16]), ([-2 ** 31 - 1], [1], None)):
        with pytest.raises(ValueError, match="32 bits"):
            cache.copy_pages(src, dst, tokens)
    cache.copy_pages([0, 1], [2, 3], [5, 32])
    cache.copy_pages([0], [np.int64(2)])
    cache.copy_pages([], [])
    assert calls == [([0, 1], [2, 3], [5, 32]), ([0], [2], None), ([], [], None)]


def test_blocks_of_a_model_share_one_rope_table():
    from types import SimpleNamespace
    from jax4j_b200.decoder import DecoderBlock
    from jax4j_b200.kv8 import PageTable, rope_table
    cache = FakeCache(9, 16)
    cache.head_dim = 128
    t = PageTable(cache, 2, 70)
    blocks = [DecoderBlock(None, SimpleNamespace(), theta=theta) for theta in (10000.0, 10000.0, 500.0)]
    tables = [b._rope_table(t) for b in blocks]
    assert tables[0] is tables[1] and tables[0] is blocks[0]._rope_table(t)
    for b, got in zip(blocks, tables):
        assert torch.equal(got, rope_table(80, 128, b.theta))
