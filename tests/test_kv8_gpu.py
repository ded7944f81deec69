"""GPU parity of the 8-bit paged KV cache's operators against the float64 oracle (oracle/kv8.py).

Bars, derived from the arithmetic:
  - append: rotations are two products and one sum, each rounded in f32, as numpy's float32 does
    them; everything after is exact or rounded by the format, so codes, scales and f32 queries are
    equal bit for bit.
  - decode: scores carry f32 rounding (|s| up to ~16 here: 16 * 2^-20 in the exponent), the second
    product f32 rounding: normwise 3e-5. A bf16 output adds half a unit, 2^-9 of the value.
  - prefill: f16 probabilities (2^-11 each) and f16 queries where they come as f32 (2^-11 of a
    score): the engine's tensor-core bar, normwise 1e-2.
  - copies: equal.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DECODE_BAR, PREFILL_BAR = 3e-5, 1e-2


def normwise(got, ref):
    return float(np.abs(np.asarray(got, np.float64) - ref).max() / max(np.abs(ref).max(), 1e-30))


def to_f8(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.float32)).cuda().to(torch.float8_e4m3fn)


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def make_pool(rng, pages, kv, page, dim):
    """Random (codes, scales) of one layer, blocks of different scales."""
    from oracle.kv8 import BLOCK, e4m3, scale_of
    x = rng.standard_normal((pages, kv, page // BLOCK, BLOCK, dim)) * 10.0 ** rng.uniform(-1, 1, (pages, kv, page // BLOCK, 1, 1))
    s = np.vectorize(scale_of)(np.abs(x).max((-1, -2)))
    return e4m3(x / s[..., None, None]).reshape(pages, kv, page, dim), s


class Pool:
    """A layer's cache on the host and the device, and sequences of given lengths on random pages.
    Everything that no sequence holds is NaN: unused pages, slots past a length, their scales."""

    def __init__(self, rng, lengths, kv, page, dim, spare=2, layers=1, layer=0, room=0):
        from jax4j_b200.kv8 import Kv8Cache
        mapped = [-(-(n + room) // page) for n in lengths]
        pages = sum(mapped) + spare
        self.k, self.ks = make_pool(rng, pages, kv, page, dim)
        self.v, self.vs = make_pool(rng, pages, kv, page, dim)
        order = rng.permutation(pages)
        self.table = np.full((len(lengths), max(1, max(mapped))), -1)
        at = 0
        for b, m in enumerate(mapped):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.lengths = list(lengths)
        self.kv, self.page, self.dim = kv, page, dim
        codes = [np.full(self.k.shape, np.nan) for _ in range(2)]
        for b, n in enumerate(lengths):
            for j0 in range(0, n, page):
                pg, m = self.table[b, j0 // page], min(page, n - j0)
                for dst, src in zip(codes, (self.k, self.v)):
                    dst[pg, :, :m] = src[pg, :, :m]
        self.codes = codes
        self.cache = Kv8Cache(pages, kv, page, dim, layers)
        self.layer = layer
        for t, c in ((self.cache.k, codes[0]), (self.cache.v, codes[1])):
            t[layer].view(torch.uint8).copy_(to_f8(c).view(torch.uint8))
        self.cache.k_scale[layer] = torch.from_numpy(self.ks).float()
        self.cache.v_scale[layer] = torch.from_numpy(self.vs).float()

    def unmap(self, b, pages):
        self.table[b, pages] = -1

    def reference(self, q, b, first_pos, window, sinks, scale=None):
        from oracle.kv8 import attention, values
        return attention(np.asarray(q, np.float64), values(self.k, self.ks), values(self.v, self.vs), self.table[b], self.lengths[b], first_pos,
                         window, sinks, scale)


DECODE = [
    # lengths, heads, kv_heads, dim, page, window, sinks
    ([0, 1, 2, 15, 16, 17, 100, 0], 4, 4, 128, 32, 0, 0),
    ([1], 1, 1, 64, 16, 0, 0),
    ([33, 200, 7], 8, 2, 128, 64, 0, 0),
    ([33, 200, 7], 16, 2, 64, 48, 0, 0),
    ([129, 64], 15, 3, 128, 16, 0, 0),       # 5 heads a group
    ([300, 77, 1], 24, 2, 128, 128, 0, 0),   # 12 heads a group: two runs
    ([3001], 8, 1, 64, 64, 0, 0),            # one row on many CTAs
    ([5000, 3, 0, 1234], 2, 1, 128, 32, 0, 0),
    ([100, 400, 31, 0], 6, 2, 128, 32, 40, 0),
    ([100, 400, 31, 50], 6, 2, 64, 16, 40, 5),
    ([257, 90], 4, 1, 128, 64, 1, 1),
    ([1000, 999], 4, 4, 128, 32, 100, 37),
    ([500], 4, 4, 128, 32, 600, 4),          # a window longer than the sequence
    ([70, 90], 4, 2, 128, 32, 20, 60),       # sinks that reach the window
]


@pytest.mark.parametrize("lengths,heads,kv,dim,page,window,sinks", DECODE)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_matches_float64(lengths, heads, kv, dim, page, window, sinks, dtype):
    rng = np.random.default_rng(len(lengths) + heads + dim + window)
    pool = Pool(rng, lengths, kv, page, dim)
    q = torch.from_numpy(rng.standard_normal((len(lengths), heads, dim)).astype(np.float32)).cuda().to(dtype)
    out = pool.cache.attention_decode(q, ints(pool.table), ints(lengths), window=window, sinks=sinks)
    assert out.dtype == dtype
    full = pool.cache.attention_decode(q, ints(pool.table), ints(lengths), window=window, sinks=sinks, out_dtype=torch.float32)
    assert torch.equal(out, full.to(dtype))
    qh, got = q.double().cpu().numpy(), full.cpu().numpy()
    ref = np.stack([pool.reference(qh[b:b + 1], b, n - 1, window, sinks)[0] for b, n in enumerate(lengths)])
    assert np.all(np.isfinite(got))
    assert not got[np.array(lengths) == 0].any()
    assert normwise(got, ref) <= DECODE_BAR


def test_decode_takes_strided_queries_tables_and_other_output_types():
    rng = np.random.default_rng(5)
    lengths, heads, kv, dim = [40, 9, 120], 4, 2, 128
    pool = Pool(rng, lengths, kv, 32, dim, layers=3, layer=2)
    wide = torch.from_numpy(rng.standard_normal((3, (heads + 2 * kv) * dim)).astype(np.float32)).cuda()
    q = wide[:, :heads * dim].unflatten(1, (heads, dim))  # rows further apart than heads * dim
    table = torch.full((3, pool.table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    table[:, :pool.table.shape[1]] = ints(pool.table)
    ref = np.stack([pool.reference(q.double().cpu().numpy()[b:b + 1], b, n - 1, 0, 0, 0.2)[0] for b, n in enumerate(lengths)])
    out = torch.full((3, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    got = pool.cache.attention_decode(q, table[:, :pool.table.shape[1]], ints(lengths), scale=0.2, layer=2, out=out)
    assert got is out
    full = pool.cache.attention_decode(q, table, ints(lengths), scale=0.2, layer=2)  # entries past the pages are not pages
    assert normwise(full.cpu().numpy(), ref) <= DECODE_BAR
    assert torch.equal(out, full.to(torch.bfloat16))


def test_decode_skips_unmapped_pages_and_gives_zeros_where_nothing_is_seen():
    rng = np.random.default_rng(6)
    lengths, heads, kv, dim, page = [300, 100, 64], 4, 2, 64, 32
    pool = Pool(rng, lengths, kv, page, dim)
    pool.unmap(0, [1, 4, 9])
    pool.unmap(1, slice(None))
    q = torch.from_numpy(rng.standard_normal((3, heads, dim)).astype(np.float32)).cuda()
    got = pool.cache.attention_decode(q, ints(pool.table), ints(lengths)).double().cpu().numpy()
    ref = np.stack([pool.reference(q.double().cpu().numpy()[b:b + 1], b, n - 1, 0, 0)[0] for b, n in enumerate(lengths)])
    assert not got[1].any()
    assert normwise(got, ref) <= DECODE_BAR
    # a length past the mapped pages sees what is mapped
    short = pool.cache.attention_decode(q, ints(pool.table[:, :2]), ints(lengths)).double().cpu().numpy()
    pool.table = pool.table[:, :2]
    ref = np.stack([pool.reference(q.double().cpu().numpy()[b:b + 1], b, n - 1, 0, 0)[0] for b, n in enumerate(lengths)])
    assert normwise(short, ref) <= DECODE_BAR


def test_decode_queries_and_values_of_extreme_magnitudes():
    """Large and tiny queries (against tiny and large keys) and value blocks whose scales differ by
    2^30: the f16 operands must not overflow or lose them."""
    rng = np.random.default_rng(7)
    lengths, heads, dim = [90], 2, 128
    for big in (1e20, 1e-20):
        pool = Pool(rng, lengths, 2, 32, dim)
        up = 2.0 ** np.round(-np.log2(big))
        pool.ks *= up
        pool.vs[:, :, 0] *= 2.0 ** 30
        pool.cache.k_scale[0] = torch.from_numpy(pool.ks).float()
        pool.cache.v_scale[0] = torch.from_numpy(pool.vs).float()
        q = (rng.standard_normal((1, heads, dim)) * big).astype(np.float32)
        got = pool.cache.attention_decode(torch.from_numpy(q).cuda(), ints(pool.table), ints(lengths)).double().cpu().numpy()
        assert normwise(got, pool.reference(q, 0, 89, 0, 0)[None, 0]) <= DECODE_BAR


def test_decode_carries_nan_of_what_it_sees():
    rng = np.random.default_rng(8)
    pool = Pool(rng, [40, 40], 1, 32, 64)
    pool.cache.v.view(torch.uint8)[0, int(pool.table[1, 0]), 0, 3] = 0x7f  # a NaN value among the seen
    q = torch.randn(2, 2, 64, device="cuda")
    got = pool.cache.attention_decode(q, ints(pool.table), ints([40, 40]))
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all()


def test_decode_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(9)
    lengths = [200, 30]
    pool = Pool(rng, lengths, 2, 32, 128)
    q = torch.from_numpy(rng.standard_normal((2, 4, 128)).astype(np.float32)).cuda()
    table, n = ints(pool.table), ints(lengths)
    want = pool.cache.attention_decode(q, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.cache.attention_decode(q, table, n)
    side.synchronize()
    assert torch.equal(want, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pool.cache.attention_decode(q, table, n)
    for m in ([200, 30], [0, 1], [33, 16]):  # the captured call follows the device's lengths
        n.copy_(ints(m))
        graph.replay()
        assert torch.equal(out, pool.cache.attention_decode(q, table, n)), m


def test_decode_is_deterministic():
    rng = np.random.default_rng(10)
    pool = Pool(rng, [4000, 17, 900], 2, 64, 128)
    q = torch.from_numpy(rng.standard_normal((3, 8, 128)).astype(np.float32)).cuda()
    a = pool.cache.attention_decode(q, ints(pool.table), ints(pool.lengths))
    for _ in range(5):
        assert torch.equal(a, pool.cache.attention_decode(q, ints(pool.table), ints(pool.lengths)))


PREFILL = [
    # (past, new) of each sequence, heads, kv_heads, dim, page, window, sinks
    ([(0, 1), (0, 64), (5, 3)], 2, 2, 128, 32, 0, 0),
    ([(0, 130)], 1, 1, 64, 16, 0, 0),
    ([(100, 0), (33, 70), (0, 0), (1, 1)], 8, 2, 128, 64, 0, 0),
    ([(200, 45), (16, 129)], 10, 2, 128, 48, 0, 0),
    ([(0, 300)], 12, 1, 64, 128, 0, 0),
    ([(130, 150), (0, 40)], 4, 2, 128, 32, 50, 0),
    ([(130, 150), (0, 40)], 4, 2, 64, 32, 50, 7),
    ([(0, 400)], 2, 1, 128, 16, 33, 130),
    ([(7, 260)], 4, 4, 128, 64, 1, 0),
]


def prefill_inputs(rng, spans, heads, kv, dim, page, dtype):
    pool = Pool(rng, [m + n for m, n in spans], kv, page, dim)
    offsets = np.cumsum([0] + [n for _, n in spans])
    q = torch.from_numpy(rng.standard_normal((offsets[-1], heads, dim)).astype(np.float32)).cuda().to(dtype)
    return pool, offsets, q


@pytest.mark.parametrize("spans,heads,kv,dim,page,window,sinks", PREFILL)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_matches_float64(spans, heads, kv, dim, page, window, sinks, dtype):
    rng = np.random.default_rng(sum(n for _, n in spans) + heads + dim + window)
    pool, offsets, q = prefill_inputs(rng, spans, heads, kv, dim, page, dtype)
    out = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks)
    got, qh = out.double().cpu().numpy(), q.double().cpu().numpy()
    assert np.all(np.isfinite(got))
    for b, (past, n) in enumerate(spans):
        if n:
            rows = slice(offsets[b], offsets[b + 1])
            assert normwise(got[rows], pool.reference(qh[rows], b, past, window, sinks)) <= PREFILL_BAR, b


def test_prefill_unmapped_pages_strides_types_and_empty_rows():
    rng = np.random.default_rng(21)
    spans, heads, kv, dim, page = [(96, 100), (40, 30)], 6, 2, 128, 32
    pool, offsets, q = prefill_inputs(rng, spans, heads, kv, dim, page, torch.float32)
    pool.unmap(0, [0, 2, 4])
    pool.unmap(1, slice(None))
    wide = torch.zeros(q.shape[0], heads + 3, dim, device="cuda")
    wide[:, :heads] = q
    got = pool.cache.attention_prefill(wide[:, :heads], ints(offsets), ints(pool.table), ints(pool.lengths), window=40, sinks=3,
                                       out_dtype=torch.bfloat16)
    assert got.dtype == torch.bfloat16
    got = got.double().cpu().numpy()
    qh = q.double().cpu().numpy()
    assert normwise(got[:100], pool.reference(qh[:100], 0, 96, 40, 3)) <= PREFILL_BAR
    assert not got[100:].any()


def test_prefill_agrees_with_decode_on_the_last_token():
    rng = np.random.default_rng(22)
    spans = [(0, 77), (300, 20), (10, 1)]
    pool, offsets, q = prefill_inputs(rng, spans, 8, 2, 128, 32, torch.float32)
    full = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths))
    last = torch.tensor(offsets[1:] - 1, device="cuda")
    one = pool.cache.attention_decode(q[last], ints(pool.table), ints(pool.lengths))
    assert normwise(full[last].cpu().numpy(), one.double().cpu().numpy()) <= PREFILL_BAR


APPEND = [
    # (start, new) of each sequence, heads, kv_heads, dim, page
    ([(0, 1)], 1, 1, 64, 16),
    ([(0, 16), (16, 16), (5, 11)], 2, 2, 128, 32),
    ([(3, 1), (15, 1), (16, 1), (40, 1), (0, 1)], 8, 2, 128, 32),
    ([(7, 50), (0, 0), (64, 3), (31, 33)], 6, 3, 64, 48),
    ([(0, 200), (190, 7)], 4, 4, 128, 64),
]


@pytest.mark.parametrize("spans,heads,kv,dim,page", APPEND)
@pytest.mark.parametrize("louder", [False, True])
def test_append_matches_the_oracle_exactly(spans, heads, kv, dim, page, louder):
    """`louder`: the new tokens outgrow the scale of the block that they join, so its old codes are
    rescaled; otherwise they are quieter and the scale stays."""
    from jax4j_b200.kv8 import rope_table
    from oracle import kv8 as O
    rng = np.random.default_rng(sum(n for _, n in spans) + heads + dim)
    pool = Pool(rng, [m for m, _ in spans], kv, page, dim, room=max(n for _, n in spans))
    offsets = np.cumsum([0] + [n for _, n in spans])
    tokens = int(offsets[-1])
    qkv = (rng.standard_normal((tokens, (heads + 2 * kv) * dim)) * (300.0 if louder else 0.01)).astype(np.float32)
    rope = rope_table(max(m + n for m, n in spans), dim, device="cuda")
    q = pool.cache.append(torch.from_numpy(qkv).cuda(), rope, ints(pool.table), ints([m for m, _ in spans]), heads,
                          offsets=None if all(n == 1 for _, n in spans) else ints(offsets))
    cs = rope.cpu().numpy()
    x = qkv.reshape(tokens, heads + 2 * kv, dim)
    k, ks, v, vs = pool.codes[0].copy(), pool.ks.copy(), pool.codes[1].copy(), pool.vs.copy()
    want_q = np.empty((tokens, heads, dim), np.float32)
    for b, (start, n) in enumerate(spans):
        rot = np.empty((n, heads + kv, dim), np.float32)
        for i in range(n):
            rot[i] = O.rope(x[offsets[b] + i, :heads + kv], cs[start + i])
        want_q[offsets[b]:offsets[b + 1]] = rot[:, :heads]
        O.append(k, ks, rot[:, heads:].astype(np.float64), pool.table[b], start)
        O.append(v, vs, x[offsets[b]:offsets[b + 1], heads + kv:].astype(np.float64), pool.table[b], start)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(pool.cache.k_scale[0].double().cpu().numpy(), ks)
    assert np.array_equal(pool.cache.v_scale[0].double().cpu().numpy(), vs)
    assert np.array_equal(pool.cache.k[0].double().cpu().numpy(), k, equal_nan=True)
    assert np.array_equal(pool.cache.v[0].double().cpu().numpy(), v, equal_nan=True)


def test_append_token_by_token_equals_its_own_rule_and_rounds_q_to_bf16():
    from jax4j_b200.kv8 import Kv8Cache, rope_table
    from oracle import kv8 as O
    rng = np.random.default_rng(31)
    heads, kv, dim, page, n = 4, 2, 128, 32, 40
    cache = Kv8Cache(3, kv, page, dim)
    table = np.array([[2, 0]])
    rope = rope_table(n, dim, device="cuda")
    k, v = np.zeros((3, kv, page, dim)), np.zeros((3, kv, page, dim))
    ks, vs = np.zeros((3, kv, 2)), np.zeros((3, kv, 2))
    for pos in range(n):
        qkv = (rng.standard_normal((1, (heads + 2 * kv) * dim)) * 2.0 ** rng.integers(-6, 6)).astype(np.float32)
        q = cache.append(torch.from_numpy(qkv).cuda(), rope, ints(table), ints([pos]), heads, q_dtype=torch.bfloat16)
        x = qkv.reshape(heads + 2 * kv, dim)
        rot = O.rope(x[:heads + kv], rope[pos].cpu().numpy())
        assert torch.equal(q[0].cpu(), torch.from_numpy(rot[:heads]).to(torch.bfloat16))
        O.append(k, ks, rot[None, heads:].astype(np.float64), table[0], pos)
        O.append(v, vs, x[None, heads + kv:].astype(np.float64), table[0], pos)
    assert np.array_equal(cache.k[0].double().cpu().numpy(), k) and np.array_equal(cache.k_scale[0].double().cpu().numpy(), ks)
    assert np.array_equal(cache.v[0].double().cpu().numpy(), v) and np.array_equal(cache.v_scale[0].double().cpu().numpy(), vs)


def test_append_special_values_unmapped_pages_and_positions_past_the_table():
    from jax4j_b200.kv8 import Kv8Cache, rope_table
    from oracle import kv8 as O
    dim, page = 64, 16
    cache = Kv8Cache(4, 1, page, dim)
    rope = rope_table(40, dim, device="cuda")
    qkv = torch.zeros(48, 3 * dim, device="cuda")
    qkv[:, 2 * dim:] = torch.randn(48, dim, device="cuda")
    qkv[0, 2 * dim] = float("inf")
    qkv[1, 2 * dim + 1] = -float("inf")
    qkv[2, 2 * dim + 2] = float("nan")
    table = np.array([[3, -1, 1]])
    cache.append(qkv, rope, ints(table), ints([0]), 1, offsets=ints([0, 48]))
    v, vs = np.zeros((4, 1, page, dim)), np.zeros((4, 1, 1))
    O.append(v, vs, qkv[:40, 2 * dim:].double().cpu().numpy()[:, None], table[0], 0)  # positions 40 .. 47 are past the rope table
    got = cache.v[0].double().cpu().numpy()
    assert np.array_equal(got, v, equal_nan=True)
    assert np.array_equal(cache.v_scale[0].double().cpu().numpy(), vs)
    assert np.isnan(got[3, 0, 2, 2]) and got[3, 0, 0, 0] == 448 and got[3, 0, 1, 1] == -448
    assert not cache.k[0].float().any()  # all-zero keys: zeros (some of them -0), the smallest scale
    assert cache.k_scale[0, 3, 0, 0] == 2.0 ** -120


@pytest.mark.parametrize("layers,kv,page,dim,moves", [(1, 1, 16, 64, 1), (3, 2, 48, 128, 5), (2, 8, 64, 128, 300), (5, 3, 32, 64, 40)])
@pytest.mark.parametrize("partial", [False, True])
def test_copy_pages_moves_blocks_and_scales(layers, kv, page, dim, moves, partial):
    from jax4j_b200.kv8 import Kv8Cache
    rng = np.random.default_rng(moves)
    pages = 2 * moves + 1
    cache = Kv8Cache(pages, kv, page, dim, layers)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8, device="cuda"))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.randn(t.shape, device="cuda"))
    order = rng.permutation(pages)
    src, dst = [int(x) for x in order[:moves]], [int(x) for x in order[moves:2 * moves]]
    tokens = [int(x) for x in rng.integers(0, page + 1, moves)] if partial else None
    want = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    for i in range(moves):
        nb = -(-(tokens[i] if partial else page) // 16)
        for t in want[:2]:
            t[:, dst[i], :, :16 * nb] = t[:, src[i], :, :16 * nb]
        for t in want[2:]:
            t[:, dst[i], :, :nb] = t[:, src[i], :, :nb]
    cache.copy_pages(src, dst, tokens)
    for got, t in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), want):
        assert torch.equal(got, t)


def test_refusals():
    from jax4j_b200.kv8 import Kv8Cache, rope_table
    cache = Kv8Cache(4, 2, 32, 128, layers=2)
    table, n = ints([[0, 1]]), ints([5])
    q = torch.zeros(1, 4, 128, device="cuda")
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        cache.attention_decode(torch.zeros(1, 3, 128, device="cuda"), table, n)
    with pytest.raises(ValueError, match="layer 2 outside"):
        cache.attention_decode(q, table, n, layer=2)
    with pytest.raises(ValueError, match="window and sinks"):
        cache.attention_decode(q, table, n, window=-1)
    with pytest.raises(ValueError, match="finite"):
        cache.attention_decode(q, table, n, scale=float("inf"))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        cache.attention_decode(q.half(), table, n)
    with pytest.raises(ValueError, match="int32"):
        cache.attention_decode(q, table.long(), n)
    with pytest.raises(ValueError, match="int32"):
        cache.attention_decode(q, table, n.cpu())
    with pytest.raises(ValueError, match="rows for"):
        cache.attention_decode(torch.zeros(2, 4, 128, device="cuda"), table, n)
    with pytest.raises(ValueError, match="dense within a row"):
        cache.attention_decode(torch.zeros(1, 4, 256, device="cuda")[..., ::2], table, n)
    with pytest.raises(ValueError, match="offsets"):
        cache.attention_prefill(q, n, table, n)
    rope = rope_table(8, 128, device="cuda")
    with pytest.raises(ValueError, match="qkv must be"):
        cache.append(torch.zeros(1, 7 * 128, device="cuda"), rope, table, n, 4)
    with pytest.raises(ValueError, match="one token for each sequence"):
        cache.append(torch.zeros(2, 8 * 128, device="cuda"), rope, table, n, 4)
    with pytest.raises(ValueError, match="rope must be"):
        cache.append(torch.zeros(1, 8 * 128, device="cuda"), rope[:, :32], table, n, 4)
    with pytest.raises(ValueError, match="written twice"):
        cache.copy_pages([0, 1], [2, 2])
    with pytest.raises(ValueError, match="both read and written"):
        cache.copy_pages([0, 1], [1, 2])
    with pytest.raises(ValueError, match="outside"):
        cache.copy_pages([0], [4])
    with pytest.raises(ValueError, match="tokens of a page"):
        cache.copy_pages([0], [1], [33])
    empty = cache.attention_decode(torch.zeros(0, 4, 128, device="cuda"), table[:0], n[:0])
    assert empty.shape == (0, 4, 128)
    cache.copy_pages([], [])


def test_prefill_keeps_nan_values_from_the_queries_before_them():
    """A NaN among the values makes NaN of the queries that see it, and of no other: those before it
    (causal, in the same tile) and those whose window has passed it."""
    rng = np.random.default_rng(23)
    n, window = 300, 60
    for w in (0, window):
        pool, offsets, q = prefill_inputs(rng, [(0, n)], 4, 2, 128, 32, torch.bfloat16)
        for at in (150, 290):
            pool.cache.v.view(torch.uint8)[0, int(pool.table[0, at // 32]), 1, at % 32, 7] = 0xff
        got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=w)
        bad = torch.isnan(got[:, 2:]).any(-1).cpu().numpy()  # heads of kv head 1
        pos = np.arange(n)
        sees = (pos >= 150) & ((w == 0) | (pos < 150 + window)) | (pos >= 290)
        assert np.array_equal(bad[:, 0], sees) and np.array_equal(bad[:, 1], sees)
        assert torch.isfinite(got[:, :2]).all()
        ref = pool.reference(q.double().cpu().numpy()[:150], 0, 0, w, 0)
        assert normwise(got[:150].double().cpu().numpy(), ref) <= PREFILL_BAR


@pytest.mark.parametrize("spans", [[(0, 1)] * 3, [(1000, 1), (0, 500), (3, 2)], [(0, 1300)], [(31, 1), (0, 0), (500, 600), (7, 257), (0, 256), (0, 255)]])
def test_prefill_many_items_and_tiles(spans):
    """Enough rows for several items of 256 a sequence, and for CTAs that take more than one."""
    rng = np.random.default_rng(sum(n for _, n in spans))
    pool, offsets, q = prefill_inputs(rng, spans, 24, 8, 64, 32, torch.bfloat16)
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths)).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    for b, (past, n) in enumerate(spans):
        for i in sorted({0, n // 3, n - 1} if n else ()):
            row = offsets[b] + i
            assert normwise(got[row], pool.reference(qh[row:row + 1], b, past + i, 0, 0)[0]) <= PREFILL_BAR, (b, i)


def test_decoder_block_on_the_paged_cache(backend):
    """Prompts in chunks, a fork, a window that frees pages, then decode steps, through DecoderBlock.
    The engine's cache holds the float64 oracle's keys and values within the format's rounding (and
    the projections' bar); attention over what it holds and the rest of the block are the oracle's,
    at the block's bars: 1e-2 for prefill, 1e-4 for decode."""
    from jax4j_b200.decoder import DecoderBlock, DecoderWeights
    from jax4j_b200.kv8 import Kv8Cache, PageTable
    from jax4j_b200.prng import PrngKey
    from oracle import kv8 as O
    from oracle.decoder import Block, rope
    d, heads, ffn, window, sinks = 256, 2, 512, 48, 5
    w = DecoderWeights.random(backend, d, heads, ffn, PrngKey.of(7), keep_blobs=True)
    ref = Block({k: v.cpu().numpy() for k, v in w.blobs.items()}, d, heads, ffn, backend.download(w.g_attn), backend.download(w.g_ffn))
    block, rng = DecoderBlock(backend, w), np.random.default_rng(41)
    cache = Kv8Cache(24, heads, 32, 128)
    pages = PageTable(cache, 4, 300)

    def check(x, counts, out, bar):
        q, k, v = ref.qkv(x)
        kh, vh = (O.values(c[0].double().cpu().numpy(), s[0].double().cpu().numpy()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        attn, row = np.zeros((len(x), heads, 128)), 0
        for slot, n in enumerate(counts):
            first = pages.lengths[slot] - n
            pos = np.broadcast_to(first + np.arange(n)[:, None], (n, heads))
            rows = slice(row, row + n)
            qr, kr = rope(q[rows], pos, 10000.0), rope(k[rows], pos, 10000.0)
            for i in range(n):
                page, at = pages.pages[slot][(first + i) // 32], (first + i) % 32
                for got, want, scales in ((kh[page, :, at], kr[i], cache.k_scale), (vh[page, :, at], v[rows][i], cache.v_scale)):
                    step = np.maximum(np.abs(want) * 2.0 ** -4, scales[0, page, :, at // 16].cpu().numpy()[:, None] * 2.0 ** -9)
                    assert np.all(np.abs(got - want) <= step + bar * np.abs(want).max())
            attn[rows] = O.attention(qr, kh, vh, pages.pages[slot], pages.lengths[slot], first, window, sinks)
            row += n
        assert normwise(out, ref.finish(x, attn.reshape(len(x), d))) <= bar

    for counts in ([37, 0, 70, 0], [5, 16, 1, 0], [0, 100, 0, 0]):
        x = rng.standard_normal((sum(counts), d)).astype(np.float32)
        out = backend.download(block.prefill_paged(backend.upload(x, x.shape), pages, counts, window, sinks, precision=2))
        check(x, counts, out, 1e-2)
    pages.fork(1, [3])
    for step in range(4):
        x = rng.standard_normal((4, d)).astype(np.float32)
        out = backend.download(block.decode_paged(backend.upload(x, x.shape), pages, window, sinks))
        check(x, [1] * 4, out, 1e-4)
        if step == 1:
            assert pages.trim(window, sinks) > 0
        if step == 2:
            pages.release(0)
            assert pages.compact() >= 0
    with pytest.raises(ValueError, match="rows for"):
        block.decode_paged(backend.upload(np.zeros((3, d), np.float32), (3, d)), pages)


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("window", [0, 150])
def test_prefill_maxima_that_are_outgrown_many_times(rising, window):
    """Keys that get louder (or quieter) block by block, the values the other way round: with rising
    keys a row's maximum moves in tile after tile, and what counts in the end lies in blocks whose
    value scale is 2^14 below the first ones'. Scores of an rms of 2^-4 to 2^2.5: the queries' f16
    (2^-12) moves the loudest by some 1e-3 and so the probabilities; these keep 11 bits down to
    2^-18, where what is lost, 2^-29 of each of a few hundred early values 2^14 times as large as the
    last, is below 1e-3 of the sum, too."""
    rng = np.random.default_rng(31 + rising)
    n, dim, page = 500, 128, 32
    pool, offsets, q = prefill_inputs(rng, [(0, n)], 4, 2, dim, page, torch.bfloat16)
    blocks = -(-n // 16)
    for j in range(blocks):
        at = (pool.table[0, j * 16 // page], slice(None), j * 16 % page // 16)
        t = j / (blocks - 1) if rising else 1 - j / (blocks - 1)
        pool.ks[at] = 2.0 ** round(-11 + 6.5 * t)
        pool.vs[at] = 2.0 ** round(-14 * t)
    pool.cache.k_scale[0] = torch.from_numpy(pool.ks).float()
    pool.cache.v_scale[0] = torch.from_numpy(pool.vs).float()
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, out_dtype=torch.float32)
    ref = pool.reference(q.double().cpu().numpy(), 0, 0, window, 0)
    for rows in (slice(0, 100), slice(100, 300), slice(300, n), slice(n - 1, n)):
        assert normwise(got[rows].double().cpu().numpy(), ref[rows]) <= PREFILL_BAR, rows


def test_prefill_of_infinite_scores():
    """Queries so large that scores overflow: rows of infinities are NaN or finite, and never touch
    other rows."""
    rng = np.random.default_rng(33)
    pool, offsets, q = prefill_inputs(rng, [(0, 200)], 4, 2, 128, 32, torch.float32)
    loud = q.clone()
    loud[50:60] *= 1e38
    got = pool.cache.attention_prefill(loud, ints(offsets), ints(pool.table), ints(pool.lengths))
    calm = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths))
    ref = pool.reference(q.double().cpu().numpy(), 0, 0, 0, 0)
    others = [i for i in range(200) if not 50 <= i < 60]
    assert torch.isfinite(got[others]).all()
    assert normwise(got[others].cpu().numpy(), ref[others]) <= PREFILL_BAR
    assert normwise(calm.cpu().numpy(), ref) <= PREFILL_BAR


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 20)])
def test_prefill_of_two_tiles_an_item_with_nan_and_unmapped_pages(window, sinks):
    """More rows than one tile an SM: NaN values, pages that are not there, a window and sinks, where
    two tiles of rows share the key tiles."""
    rng = np.random.default_rng(41 + window)
    spans, heads, kv, dim, page = [(0, 700), (900, 333)], 32, 8, 128, 64
    pool, offsets, q = prefill_inputs(rng, spans, heads, kv, dim, page, torch.bfloat16)
    pool.unmap(1, [1, 5, 6])
    at = 450
    pool.cache.v.view(torch.uint8)[0, int(pool.table[0, at // page]), 3, at % page, 100] = 0x7f
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks).double().cpu().numpy()
    bad = np.isnan(got).any(-1)
    pos = np.arange(700)
    sees = (pos >= at) & ((window == 0) | (pos < at + window))
    want = np.zeros_like(bad)
    want[:700, 12:16] = sees[:, None]  # the query heads of kv head 3
    assert np.array_equal(bad, want)
    qh = q.double().cpu().numpy()
    for b, (past, n) in enumerate(spans):
        ref = pool.reference(qh[offsets[b]:offsets[b + 1]], b, past, window, sinks)
        mine = got[offsets[b]:offsets[b + 1]]
        for part in (slice(0, 128), slice(128, 256), slice(256, n)):
            keep = ~want[offsets[b]:offsets[b + 1]][part]
            assert normwise(mine[part][keep], ref[part][keep]) <= PREFILL_BAR, (b, part)


def test_decode_of_two_threads_on_one_stream():
    """Threads share PyTorch's default stream and the cache: each gets its own results."""
    import threading
    rng = np.random.default_rng(51)
    pool = Pool(rng, [4000, 17, 900, 2500], 2, 64, 128)
    table = ints(pool.table)
    jobs = []
    for i in range(4):
        lengths = ints([int(n * f) for n, f in zip(pool.lengths, rng.uniform(0.1, 1, 4))])
        q = torch.from_numpy(rng.standard_normal((4, 8, 128)).astype(np.float32)).cuda()
        jobs.append((q, lengths, pool.cache.attention_decode(q, table, lengths)))
    bad = []

    def work(q, lengths, want):
        outs = [pool.cache.attention_decode(q, table, lengths) for _ in range(200)]
        torch.cuda.synchronize()
        bad.extend(i for i, o in enumerate(outs) if not torch.equal(o, want))
    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def hide_loud_values(pool, b, at, up, alone):
    """Makes the value of token `at` of sequence b 2^up times as loud as its block's scale has the
    others: with its whole block, or (`alone`) by itself, and the block's other values are then below
    the format's smallest."""
    from oracle.kv8 import BLOCK
    pg, blk = pool.table[b, at // pool.page], at % pool.page // BLOCK
    rows = slice(blk * BLOCK, (blk + 1) * BLOCK)
    pool.vs[pg, :, blk] *= 2.0 ** up
    if alone:
        keep = pool.v[pg, :, at % pool.page].copy()
        pool.v[pg, :, rows] = 0
        pool.v[pg, :, at % pool.page] = keep
    codes = to_f8(pool.v[pg])
    pool.cache.v[pool.layer, int(pg)].view(torch.uint8).copy_(codes.view(torch.uint8))
    pool.cache.v_scale[pool.layer, int(pg)] = torch.from_numpy(pool.vs[pg]).float()


def quiet_keys(pool):
    """Scores near zero, so that every seen token counts."""
    pool.ks *= 2.0 ** np.round(np.log2(0.05) - np.log2(np.abs(pool.k).max((-1, -2)).reshape(pool.ks.shape[0], pool.ks.shape[1], 1) * pool.ks))
    pool.cache.k_scale[pool.layer] = torch.from_numpy(pool.ks).float()


@pytest.mark.parametrize("up,alone", [(24, False), (24, True), (40, False), (40, True)])
@pytest.mark.parametrize("heads,kv,dim,window,sinks", [(2, 1, 64, 0, 0), (8, 2, 128, 70, 0), (8, 2, 128, 70, 21), (32, 16, 64, 90, 5), (32, 32, 128, 0, 0)])
def test_prefill_rows_do_not_feel_loud_values_they_do_not_see(heads, kv, dim, window, sinks, up, alone):
    """f16 probabilities are weighed by the largest value scale that a row sees: one that it does not
    see may not push them out of f16's range. Every row by itself, those just before a loud token in
    its own block, too."""
    rng = np.random.default_rng(heads + dim + window + up)
    n = 420
    pool, offsets, q = prefill_inputs(rng, [(0, n)], heads, kv, dim, 32, torch.float32)
    quiet_keys(pool)
    for at in (23, 201, 333):
        hide_loud_values(pool, 0, at, up, alone)
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks).double().cpu().numpy()
    rows = np.unique(np.concatenate([np.arange(0, n, 37), np.arange(16, 40), np.arange(190, 225), np.arange(200 + 60, 200 + 95), np.arange(320, 345), [n - 1]]))
    qh = q.double().cpu().numpy()
    for i in rows:
        want = pool.reference(qh[i:i + 1], 0, i, window, sinks)[0]
        assert normwise(got[i], want) <= PREFILL_BAR, i


@pytest.mark.parametrize("up,alone", [(24, False), (28, True), (40, False), (40, True), (60, True)])
@pytest.mark.parametrize("heads,kv,dim,window,sinks", [(4, 2, 64, 0, 0), (6, 2, 128, 70, 0), (6, 2, 64, 70, 21), (8, 8, 128, 90, 5)])
def test_decode_does_not_feel_loud_values_it_does_not_see(heads, kv, dim, window, sinks, up, alone):
    """Loud values just past the length (what the page held before), just before the window and just
    behind the sinks, in blocks that are seen in part."""
    rng = np.random.default_rng(heads + dim + window + up)
    lengths = [100, 417, 31, 50, 2001, 7]
    pool = Pool(rng, lengths, kv, 32, dim, room=16)
    quiet_keys(pool)
    for b, n in enumerate(lengths):
        for at in [n] + ([n - window - 1, sinks] if window and n > window + sinks else []):
            hide_loud_values(pool, b, at, up, alone)
    q = torch.from_numpy(rng.standard_normal((len(lengths), heads, dim)).astype(np.float32)).cuda()
    table = ints(pool.table)
    for rows in (slice(0, len(lengths)), slice(0, 2), slice(2, 4)):  # shared out, and by a CTA each
        width = max(-(-n // 32) for n in lengths[rows])
        got = pool.cache.attention_decode(q[rows], table[rows, :width], ints(lengths[rows]), window=window, sinks=sinks).double().cpu().numpy()
        for i, b in enumerate(range(len(lengths))[rows]):
            want = pool.reference(q[b:b + 1].double().cpu().numpy(), b, lengths[b] - 1, window, sinks)[0]
            assert normwise(got[i], want) <= DECODE_BAR, b


@pytest.mark.parametrize("up,alone", [(28, False), (40, True)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_in_shares_does_not_feel_loud_values_it_does_not_see(dim, up, alone):
    """As above, with enough rows for each warp to have many blocks of one."""
    rng = np.random.default_rng(dim + up)
    kv, window, sinks = 16, 1000, 6
    lengths = [1300 + 13 * b for b in range(24)]
    pool = Pool(rng, lengths, kv, 32, dim, room=16)
    quiet_keys(pool)
    for b, n in enumerate(lengths):
        for at in (n, n - window - 1, sinks):
            hide_loud_values(pool, b, at, up, alone)
    q = torch.from_numpy(rng.standard_normal((len(lengths), kv, dim)).astype(np.float32)).cuda()
    got = pool.cache.attention_decode(q, ints(pool.table), ints(lengths), window=window, sinks=sinks).double().cpu().numpy()
    for b in range(0, len(lengths), 8):
        want = pool.reference(q[b:b + 1].double().cpu().numpy(), b, lengths[b] - 1, window, sinks)[0]
        assert normwise(got[b], want) <= DECODE_BAR, b


WILD = [2 ** 31 - 1, 2 ** 31 - 70, 2 ** 30 + 5, -1, -2 ** 31]


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 7)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_lengths_past_what_a_table_holds(dim, window, sinks):
    """Any length ends at once: past the table's last page there is nothing to walk over."""
    rng = np.random.default_rng(61)
    lengths, heads = [90, 64, 128, 33, 96], 4
    pool = Pool(rng, lengths, 2, 32, dim)
    pool.table[2:] = -1  # what a wild length sees: the pages of the first, whole, and none of its own
    pool.table[2] = pool.table[1]
    full = int((pool.table[1] >= 0).sum()) * 32
    q = torch.from_numpy(rng.standard_normal((5, heads, dim)).astype(np.float32)).cuda()
    for wild in WILD:
        n = [90, 64, wild, wild, 0]
        for width in (pool.table.shape[1], 40):  # by a CTA each, and shared out
            table = torch.full((5, width), -1, dtype=torch.int32, device="cuda")
            table[:, :pool.table.shape[1]] = ints(pool.table)
            got = pool.cache.attention_decode(q, table, ints(n), window=window, sinks=sinks).double().cpu().numpy()
            for b in (0, 1):
                assert normwise(got[b], pool.reference(q[b:b + 1].double().cpu().numpy(), b, n[b] - 1, window, sinks)[0]) <= DECODE_BAR
            assert not got[3:].any()
            if wild < 0:
                assert not got[2].any()
            else:  # the sinks, if there is a window: that one lies far past the table
                pool.lengths[2] = sinks if window else full
                assert normwise(got[2], pool.reference(q[2:3].double().cpu().numpy(), 2, pool.lengths[2] - 1, 0, 0)[0]) <= DECODE_BAR


@pytest.mark.parametrize("heads,kv", [(4, 2), (32, 32)])
def test_prefill_and_append_of_wild_lengths_and_offsets(heads, kv):
    """Sequences whose arrays make sense keep their results next to ones whose arrays do not, whose
    rows lie apart from theirs."""
    from jax4j_b200.kv8 import rope_table
    rng = np.random.default_rng(62)
    dim, page = 64, 32
    pool = Pool(rng, [70, 300, 60, 60], kv, page, dim, room=64)
    q = torch.from_numpy(rng.standard_normal((200, heads, dim)).astype(np.float32)).cuda()
    rope = rope_table(400, dim, device="cuda")
    qkv = torch.from_numpy(rng.standard_normal((200, (heads + 2 * kv) * dim)).astype(np.float32)).cuda()
    qh = q.double().cpu().numpy()
    ref = [pool.reference(qh[:70], 0, 0, 0, 0), pool.reference(qh[70:150], 1, 220, 0, 0)]
    codes = [t.clone() for t in (pool.cache.k.view(torch.uint8), pool.cache.v.view(torch.uint8))]
    for wild in WILD:
        for offsets in ([0, 70, 150, wild, -3], [0, 70, 150, 2 ** 31 - 1, -2 ** 31], [0, 70, 150, 200, 10 ** 9]):
            got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints([70, 300, wild, wild])).double().cpu().numpy()
            for rows, want in zip((slice(0, 70), slice(70, 150)), ref):
                assert normwise(got[rows], want) <= PREFILL_BAR
            starts = [70, 300, wild, wild]
            out = pool.cache.append(qkv, rope, ints(pool.table), ints(starts), heads, offsets=ints(offsets))
            alone = pool.cache.append(qkv, rope, ints(pool.table[:2]), ints(starts[:2]), heads, offsets=ints(offsets[:3]))
            assert torch.equal(out[:150], alone[:150])
            for b in (2, 3):  # nothing was written to their pages
                for t, before in zip((pool.cache.k, pool.cache.v), codes):
                    pages = torch.from_numpy(pool.table[b][pool.table[b] >= 0]).cuda()
                    assert torch.equal(t.view(torch.uint8)[0, pages], before[0, pages])


@pytest.mark.parametrize("spans,heads,kv,dim", [([(0, 300), (200, 40)], 4, 2, 64), ([(0, 300), (200, 40)], 8, 2, 128), ([(0, 700)], 32, 32, 128), ([(0, 1)] * 3, 2, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_keeps_eleven_bits(spans, heads, kv, dim, dtype):
    """What the operands' 11 bits leave, in the mean: a probability is off by some 0.41 2^-11 of itself,
    and where queries come as f32, a score by 0.41 2^-11 of its rms S (each product of its sum by
    as much of itself, signs at random). With values of random signs the result is then off by
    0.41 2^-11 sqrt(1 + S^2) of its rms; the bar is 2.4 times that. Queries or probabilities of 8
    bits would be 8 times off."""
    rng = np.random.default_rng(71 + dim)
    pool, offsets, q = prefill_inputs(rng, spans, heads, kv, dim, 32, dtype)
    pool.ks *= 2.0 ** np.round(1 - np.log2(np.sqrt((pool.k ** 2).mean((-1, -2))).reshape(*pool.ks.shape[:2], 1) * pool.ks))  # S about 2
    pool.vs[:] = 2.0 ** -8
    pool.cache.k_scale[0], pool.cache.v_scale[0] = torch.from_numpy(pool.ks).float(), torch.from_numpy(pool.vs).float()
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), out_dtype=torch.float32).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    kh = pool.k * np.repeat(pool.ks, 16, axis=2)[..., None]
    rms = float(np.sqrt((kh ** 2).mean() * (qh ** 2).mean())) if dtype is torch.float32 else 0.0
    assert rms < 4
    off, of = 0.0, 0.0
    for b, (past, n) in enumerate(spans):
        want = pool.reference(qh[offsets[b]:offsets[b + 1]], b, past, 0, 0)
        off += ((got[offsets[b]:offsets[b + 1]] - want) ** 2).sum()
        of += (want ** 2).sum()
    assert np.sqrt(off / of) <= 2.0 ** -11 * np.sqrt(1 + rms ** 2)


def test_decoder_block_gives_prefill_the_queries_as_append_rotated_them(backend, monkeypatch):
    """f32, which the kernel rounds to 11 bits: no type in between that holds fewer."""
    from jax4j_b200.decoder import DecoderBlock, DecoderWeights
    from jax4j_b200.kv8 import Kv8Cache, PageTable
    from jax4j_b200.prng import PrngKey
    cache = Kv8Cache(8, 2, 32, 128)
    pages, made, used = PageTable(cache, 2, 100), [], []
    append, attention = cache.append, cache.attention_prefill
    monkeypatch.setattr(cache, "append", lambda *a, **k: made.append(append(*a, **k)) or made[-1])
    monkeypatch.setattr(cache, "attention_prefill", lambda q, *a, **k: used.append(q) or attention(q, *a, **k))
    block = DecoderBlock(backend, DecoderWeights.random(backend, 256, 2, 512, PrngKey.of(3)))
    x = np.random.default_rng(1).standard_normal((50, 256)).astype(np.float32)
    block.prefill_paged(backend.upload(x, x.shape), pages, [20, 30])
    assert used[0] is made[0] and used[0].dtype == torch.float32


def test_a_fork_reads_as_its_parent_at_once():
    from jax4j_b200.kv8 import Kv8Cache, PageTable, rope_table
    torch.manual_seed(5)
    cache = Kv8Cache(12, 2, 16, 64)
    pages = PageTable(cache, 3, 100)
    starts, lengths, offsets = pages.extend([40, 0, 20])
    cache.append(torch.randn(60, 8 * 64, device="cuda"), rope_table(100, 64, device="cuda"), pages.table, starts, 4, offsets)
    pages.fork(0, [1])
    q = torch.randn(1, 4, 64, device="cuda").expand(3, 4, 64).contiguous()
    out = cache.attention_decode(q, pages.table, ints(pages.lengths))
    assert torch.equal(out[0], out[1]) and out[0].any()
    pages.release(0)
    assert pages.compact() > 0
    again = cache.attention_decode(q, pages.table, ints(pages.lengths))
    assert torch.equal(again[1], out[1]) and torch.equal(again[2], out[2]) and not again[0].any()


def test_decoder_block_decodes_only_active_slots(backend):
    """Idle slots take no pages and keep their sequences; the active ones get what they would get by
    themselves."""
    from jax4j_b200.decoder import DecoderBlock, DecoderWeights
    from jax4j_b200.kv8 import Kv8Cache, PageTable
    from jax4j_b200.prng import PrngKey
    block = DecoderBlock(backend, DecoderWeights.random(backend, 256, 2, 512, PrngKey.of(3)))
    rng = np.random.default_rng(81)
    prompt, steps = rng.standard_normal((50, 256)).astype(np.float32), rng.standard_normal((20, 4, 256)).astype(np.float32)
    outs = []
    for slots, counts, active in ((4, [20, 30, 0, 0], [True, False, False, True]), (2, [20, 0], None)):
        pages = PageTable(Kv8Cache(8, 2, 16, 128), slots, 64)
        x = prompt[:sum(counts)]
        block.prefill_paged(backend.upload(x, x.shape), pages, counts)
        for step in steps:
            x = step if active else step[[0, 3]]
            out = backend.download(block.decode_paged(backend.upload(x, x.shape), pages, active=active))
        outs.append(out)
        if active:
            assert pages.lengths == [40, 30, 0, 20] and [len(p) for p in pages.pages] == [3, 2, 0, 2]
            pages.fork(0, [2])  # an idle slot is still without a sequence
    assert normwise(outs[0][[0, 3]], outs[1].astype(np.float64)) <= 1e-4
    with pytest.raises(ValueError, match="3 entries for 4 slots"):
        block.decode_paged(backend.upload(steps[0], (4, 256)), PageTable(Kv8Cache(8, 2, 16, 128), 4, 64), active=[1, 1, 1])


def test_one_row_of_any_stride():
    rng = np.random.default_rng(91)
    pool = Pool(rng, [50], 2, 32, 64)
    q = torch.from_numpy(rng.standard_normal((1, 6, 64)).astype(np.float32)).cuda()
    odd = q[0].unsqueeze(1).transpose(0, 1)
    assert odd.stride(0) == 64 and odd.is_contiguous()
    table, n = ints(pool.table), ints([50])
    assert torch.equal(pool.cache.attention_decode(odd, table, n), pool.cache.attention_decode(q, table, n))
    assert torch.equal(pool.cache.attention_prefill(odd, ints([0, 1]), table, n), pool.cache.attention_prefill(q, ints([0, 1]), table, n))


@pytest.mark.parametrize("dim", [64, 128])
def test_queries_near_the_end_of_f32(dim):
    """Queries of 2^116 against keys of as little (scores of an rms of 2): as exact as any."""
    rng = np.random.default_rng(95)
    pool = Pool(rng, [90], 2, 32, dim)
    pool.ks *= 2.0 ** np.round(1 - 114 - np.log2(np.sqrt((pool.k ** 2).mean((-1, -2))).reshape(*pool.ks.shape[:2], 1) * pool.ks))
    pool.cache.k_scale[0] = torch.from_numpy(pool.ks).float()
    q = (rng.standard_normal((90, 4, dim)) * 2.0 ** 114).astype(np.float32)
    assert np.isfinite(q).all() and np.abs(q).max() > 2.0 ** 115
    qd = torch.from_numpy(q).cuda()
    table, n = ints(pool.table), ints([90])
    got = pool.cache.attention_decode(qd[-1:], table, n).double().cpu().numpy()
    assert normwise(got[0], pool.reference(q[-1:], 0, 89, 0, 0)[0]) <= DECODE_BAR
    got = pool.cache.attention_prefill(qd, ints([0, 90]), table, n).double().cpu().numpy()
    assert normwise(got, pool.reference(q, 0, 0, 0, 0)) <= PREFILL_BAR


def repeated_pages(rng, heads, dim, page, width, n):
    """A sequence whose table names two pages over and over, and n queries at its end."""
    pool = Pool(rng, [2 * page], heads, page, dim, spare=0)
    quiet_keys(pool)
    q = torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).cuda().to(torch.bfloat16)
    return pool, q, ints(np.array(pool.table[0])[np.arange(width) % 2][None]), width * page


def test_prefill_waits_as_long_as_an_item_takes():
    """Over 2^24 tokens an item (256 rows) takes 0.3 s, longer than most waits may: the ones for a whole
    item go by the length. Its rows are what they are in a call of few items, where none waits."""
    heads, n = 16, 7680  # four items for some SMs, which is as many as are found ahead
    pool, q, table, length = repeated_pages(np.random.default_rng(97), heads, 64, 4096, 4096, n)
    got = pool.cache.attention_prefill(q, ints([0, n]), table, ints([length]))
    for i in (0, 3000, n - 1):
        one = pool.cache.attention_prefill(q[i:i + 1], ints([0, 1]), table, ints([length - n + i + 1]))  # reports a wait that gave up
        assert torch.equal(got[i], one[0]), i


def test_prefill_over_a_million_tokens():
    """The softmax is one over the two pages' tokens, each as often as it is seen. 2^16 additions to the
    tensor cores' f32, rounded toward zero, lose up to 2^-24 of the sum each in the mean: 4e-3, and the
    operands' bits 1e-3."""
    from oracle.kv8 import values
    heads, dim, page, n = 4, 128, 4096, 300
    pool, q, table, length = repeated_pages(np.random.default_rng(98), heads, dim, page, 256, n)
    got = pool.cache.attention_prefill(q, ints([0, n]), table, ints([length]), out_dtype=torch.float32).double().cpu().numpy()
    k, v = (values(c, s)[pool.table[0]].transpose(1, 0, 2, 3).reshape(heads, 2 * page, dim) for c, s in ((pool.k, pool.ks), (pool.v, pool.vs)))
    for i in (0, 130, 255, n - 1):
        seen = length - n + i + 1
        count = seen // (2 * page) + (np.arange(2 * page) < seen % (2 * page))
        w = count * np.exp(np.einsum("hkd,hd->hk", k, q[i].double().cpu().numpy()) * dim ** -0.5)
        assert normwise(got[i], np.einsum("hk,hkd->hd", w / w.sum(-1, keepdims=True), v)) <= PREFILL_BAR, i


@pytest.mark.parametrize("heads,kv,window,sinks", [(2, 2, 20, 0), (2, 2, 20, 5), (32, 32, 20, 0), (32, 32, 20, 5), (8, 2, 150, 0), (4, 4, 0, 0)])
def test_prefill_rows_do_not_feel_key_tiles_that_are_loud_throughout(heads, kv, window, sinks):
    """As above, where all blocks of a key tile are as loud and some rows see none of them."""
    rng = np.random.default_rng(heads + window + sinks)
    n, dim = 460, 64
    pool, offsets, q = prefill_inputs(rng, [(0, n)], heads, kv, dim, 32, torch.float32)
    quiet_keys(pool)
    for at in range(64, 208, 16):
        hide_loud_values(pool, 0, at, 30, False)
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    for i in np.unique(np.concatenate([np.arange(0, n, 29), np.arange(55, 72), np.arange(200, 232), np.arange(340, 364)])):
        want = pool.reference(qh[i:i + 1], 0, i, window, sinks)[0]
        assert normwise(got[i], want) <= PREFILL_BAR, i


def nan_scales_of_what_nobody_holds(pool):
    for t in (pool.cache.k_scale, pool.cache.v_scale):
        held = torch.zeros(t.shape[1], t.shape[3], dtype=torch.bool)
        for b, n in enumerate(pool.lengths):
            for blk in range(-(-n // 16)):
                held[int(pool.table[b, blk * 16 // pool.page]), blk * 16 % pool.page // 16] = True
        t[pool.layer][~held[:, None, :].expand(-1, t.shape[2], -1).cuda()] = float("nan")


def many_lengths(rng, n, most):
    """n lengths up to `most`, every fifth sequence (and the first and the last) empty."""
    return [0 if i % 5 == 0 or i == n - 1 else int(x) for i, x in enumerate(rng.integers(1, most + 1, n))]


@pytest.mark.parametrize("n,most,width,window,sinks", [(200, 60, 0, 0, 0), (200, 300, 0, 0, 0), (131, 700, 40, 90, 3), (500, 40, 0, 0, 0)])
def test_decode_of_many_sequences(n, most, width, window, sinks):
    """More sequences than a CTA's threads, whose search for a share then gives a thread several."""
    rng = np.random.default_rng(n + most)
    lengths = many_lengths(rng, n, most)
    pool = Pool(rng, lengths, 2, 32, 64)
    nan_scales_of_what_nobody_holds(pool)
    table = torch.full((n, max(width, pool.table.shape[1])), -1, dtype=torch.int32, device="cuda")
    table[:, :pool.table.shape[1]] = ints(pool.table)
    q = torch.from_numpy(rng.standard_normal((n, 4, 64)).astype(np.float32)).cuda()
    got = pool.cache.attention_decode(q, table, ints(lengths), window=window, sinks=sinks).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    assert np.isfinite(got).all() and not got[np.array(lengths) == 0].any()
    for b in range(n):
        if lengths[b]:
            assert normwise(got[b], pool.reference(qh[b:b + 1], b, lengths[b] - 1, window, sinks)[0]) <= DECODE_BAR, b


@pytest.mark.parametrize("n,heads,kv,window,sinks", [(40, 2, 1, 0, 0), (70, 8, 4, 0, 0), (70, 8, 4, 50, 7), (33, 32, 16, 0, 0)])
def test_prefill_of_many_sequences(n, heads, kv, window, sinks):
    """More sequences than a warp's lanes, past which the search for an item reads them again."""
    rng = np.random.default_rng(n + heads + window)
    new, past = many_lengths(rng, n, 150), many_lengths(rng, n, 100)[::-1]
    pool, offsets, q = prefill_inputs(rng, list(zip(past, new)), heads, kv, 64, 32, torch.float32)
    nan_scales_of_what_nobody_holds(pool)
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    assert np.isfinite(got).all()
    for b in range(n):
        for i in sorted({0, new[b] // 2, new[b] - 1} if new[b] else ()):
            row = int(offsets[b]) + i
            assert normwise(got[row], pool.reference(qh[row:row + 1], b, past[b] + i, window, sinks)[0]) <= PREFILL_BAR, (b, i)


@pytest.mark.parametrize("one", [False, True])
def test_append_of_many_sequences(one):
    from jax4j_b200.kv8 import rope_table
    from oracle import kv8 as O
    rng = np.random.default_rng(200 + one)
    n, heads, kv, dim, page = 200, 2, 1, 64, 32
    starts = many_lengths(rng, n, 40)
    new = [1] * n if one else many_lengths(rng, n, 25)[::-1]
    pool = Pool(rng, starts, kv, page, dim, room=25)
    nan_scales_of_what_nobody_holds(pool)
    pool.ks, pool.vs = (t[0].double().cpu().numpy() for t in (pool.cache.k_scale, pool.cache.v_scale))
    offsets = np.cumsum([0] + new)
    qkv = rng.standard_normal((offsets[-1], (heads + 2 * kv) * dim)).astype(np.float32)
    rope = rope_table(70, dim, device="cuda")
    q = pool.cache.append(torch.from_numpy(qkv).cuda(), rope, ints(pool.table), ints(starts), heads, offsets=None if one else ints(offsets))
    cs, x = rope.cpu().numpy(), qkv.reshape(-1, heads + 2 * kv, dim)
    k, ks, v, vs = pool.codes[0].copy(), pool.ks.copy(), pool.codes[1].copy(), pool.vs.copy()
    for b, (start, m) in enumerate(zip(starts, new)):
        rows = slice(offsets[b], offsets[b + 1])
        rot = np.stack([O.rope(x[offsets[b] + i, :heads + kv], cs[start + i]) for i in range(m)]) if m else np.empty((0, heads + kv, dim), np.float32)
        assert np.array_equal(q[rows].cpu().numpy(), rot[:, :heads]), b
        O.append(k, ks, rot[:, heads:].astype(np.float64), pool.table[b], start)
        O.append(v, vs, x[rows, heads + kv:].astype(np.float64), pool.table[b], start)
    for got, want in ((pool.cache.k_scale, ks), (pool.cache.v_scale, vs), (pool.cache.k, k), (pool.cache.v, v)):
        assert np.array_equal(got[0].double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("kv,group,dim", [(16, 7, 128), (16, 1, 64), (2, 2, 64)])
def test_prefill_past_runs_of_queries_that_see_nothing(kv, group, dim):
    """Sequences whose queries all lie before their cache (no length, or fewer tokens than queries) give
    zeros, and however many of them a CTA gets one after the other, the ones between are computed."""
    rng = np.random.default_rng(kv + group)
    spans = []  # (tokens, queries)
    for i in range(60):
        spans.append((int(rng.integers(1, 150)), int(rng.integers(1, 40))) if i % 11 == 0 or i > 56 else (0, int(rng.integers(1, 4))))
    pool = Pool(rng, [n for n, _ in spans], kv, 32, dim)
    offsets = np.cumsum([0] + [n for _, n in spans])
    q = torch.from_numpy(rng.standard_normal((offsets[-1], kv * group, dim)).astype(np.float32)).cuda()
    out = torch.full_like(q, 7.0)
    for window in (0, 2):
        got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, out=out).double().cpu().numpy()
        qh = q.double().cpu().numpy()
        for b, (m, n) in enumerate(spans):
            rows, before = slice(offsets[b], offsets[b + 1]), max(0, n - m)
            assert not got[rows][:before].any(), b
            if m:
                assert normwise(got[rows][before:], pool.reference(qh[rows][before:], b, max(0, m - n), window, 0)) <= PREFILL_BAR, b
    none = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints([0] * 60), out=out)  # also reports a wait that gave up
    assert not none.any()
    pool.cache.attention_prefill(q[:1], ints([0, 1]), ints(pool.table[:1]), ints(pool.lengths[:1]))


@pytest.mark.parametrize("heads,kv,window,sinks", [(2, 2, 0, 0), (8, 2, 0, 0), (32, 32, 0, 0), (2, 2, 100, 0), (32, 32, 100, 0), (8, 2, 100, 16), (8, 2, 100, 3), (32, 32, 100, 20)])
@pytest.mark.parametrize("at", [16, 128, 144, 256])
def test_prefill_rows_at_the_edge_of_a_loud_key_tile(heads, kv, window, sinks, at):
    """Rows that see of a key tile, loud throughout, only its first tokens or (under the window) its last
    ones, whose own values the loud ones in their blocks left as zeros."""
    rng = np.random.default_rng(heads + window + sinks + at)
    n, dim = 500, 64
    pool, offsets, q = prefill_inputs(rng, [(0, n)], heads, kv, dim, 32, torch.float32)
    quiet_keys(pool)
    pool.vs[:] = 2.0 ** -5
    pool.cache.v_scale[0] = 2.0 ** -5
    for blk in range(at, at + 128, 16):
        hide_loud_values(pool, 0, blk, 30, False)
    for lo, hi in ((at, at + 7), (at + 128 - 5, at + 128)):
        pg = int(pool.table[0, lo // 32])
        pool.v[pg, :, lo % 32:lo % 32 + hi - lo] = 0
        pool.cache.v[0, pg].view(torch.uint8).copy_(to_f8(pool.v[pg]).view(torch.uint8))
    got = pool.cache.attention_prefill(q, ints(offsets), ints(pool.table), ints(pool.lengths), window=window, sinks=sinks).double().cpu().numpy()
    qh = q.double().cpu().numpy()
    for i in list(range(at - 3, at + 12)) + (list(range(at + 118 + window, min(n, at + 132 + window)))  if window else []) + [n - 1]:
        want = pool.reference(qh[i:i + 1], 0, i, window, sinks)[0]
        assert normwise(got[i], want) <= PREFILL_BAR, i
