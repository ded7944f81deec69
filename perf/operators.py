"""Timing cases of the 8-bit paged KV cache: appending tokens, attention over the pages, page copies.

The cache holds keys and values as e4m3 codes [layers, pages, kv_heads, page, head_dim] with one power-of-two f32 scale for
each block of 16 tokens and head, [layers, pages, kv_heads, page / 16]. A sequence's pages are named by its row of a page table
(int32, -1 = unmapped). Each case is one pass through one operator:

  append    RoPE of the new tokens' queries and keys, quantisation of keys and values into their pages
  decode    one query per sequence over its cached tokens
  prefill   ragged chunks of new queries over their cached tokens, causal
  pages     copies of pages within every layer (forks of a partly filled page, compaction)

Attention takes grouped heads, a sliding window and first tokens ("sinks") that stay visible. Lengths and page counts follow
from the case alone; values and page numbers from the seed.
"""
import math

import torch

own = False

BLOCK = 16  # tokens that share a scale
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # append: one new token for each of 64 sequences of the decoder block's own shape (32 heads of 128): a decode step's write
        dict(name="append step 64", op="append", batch=64, heads=32, kv_heads=32, head_dim=128, page=64, new=1, past=2048, dtype="float32"),
        # continued prompts of odd lengths that start inside a block, grouped heads
        dict(name="append ragged chunks", op="append", batch=16, heads=32, kv_heads=8, head_dim=128, page=32, new=2047, past=1500, dtype="bfloat16", ragged=True),
        # decode: one user's short chat, grouped heads: latency
        dict(name="decode one short", op="decode", batch=1, heads=32, kv_heads=8, head_dim=128, page=64, length=517, window=0, sinks=0, dtype="float32"),
        # the decoder block's decode step: batch 64, 2048 cached tokens and the new one, 32 heads
        dict(name="decode 64x2049", op="decode", batch=64, heads=32, kv_heads=32, head_dim=128, page=64, length=2049, window=0, sinks=0, dtype="float32"),
        # a serving batch of mixed lengths with idle slots
        dict(name="decode ragged", op="decode", batch=48, heads=32, kv_heads=8, head_dim=128, page=32, length=8191, window=0, sinks=0, dtype="bfloat16", ragged=True),
        # two long documents: few rows, a long axis
        dict(name="decode long 2x131071", op="decode", batch=2, heads=32, kv_heads=8, head_dim=128, page=128, length=131071, window=0, sinks=0, dtype="float32"),
        # streaming generation: a window with sinks, pages that fell out of it freed
        dict(name="decode window", op="decode", batch=32, heads=40, kv_heads=8, head_dim=64, page=16, length=30001, window=4096, sinks=4, dtype="bfloat16"),
        # prefill: short turns of running chats over their past
        dict(name="prefill turns", op="prefill", batch=5, heads=32, kv_heads=8, head_dim=128, page=64, new=77, past=1000, window=0, sinks=0, dtype="bfloat16", ragged=True),
        # the decoder block's prefill, 8 x 2048 causal
        dict(name="prefill 8x2048", op="prefill", batch=8, heads=32, kv_heads=32, head_dim=128, page=64, new=2048, past=0, window=0, sinks=0, dtype="bfloat16"),
        # one long prompt under a window with sinks
        dict(name="prefill window 8001", op="prefill", batch=1, heads=32, kv_heads=8, head_dim=128, page=64, new=8001, past=0, window=1024, sinks=16, dtype="bfloat16"),
        # pages: compaction after a burst of short requests, every layer of a 16-layer cache
        dict(name="pages compact", op="pages", layers=16, pages=320, moves=147, kv_heads=8, head_dim=128, page=64, partial=False),
        # forking 12 beams off their prompts: only the filled blocks of each last page move
        dict(name="pages fork", op="pages", layers=8, pages=64, moves=12, kv_heads=8, head_dim=128, page=64, partial=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "pages"])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 8, 12])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 48, 64, 64, 128])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "pages":
        page_bytes = 2 * kv * page * dim
        layers = _log(rng, 1, 32)
        moves = _log(rng, 1, max(1, min(256, (300 << 20) // (layers * page_bytes))))
        return dict(op=op, layers=layers, pages=2 * moves + rng.randint(1, 9), moves=moves, kv_heads=kv, head_dim=dim, page=page,
                    partial=rng.random() < 0.5)
    shape = dict(op=op, heads=kv * group, kv_heads=kv, head_dim=dim, page=page, dtype=dtype, ragged=rng.random() < 0.6)
    if op == "decode":
        batch = _log(rng, 1, 64)
        length = _log(rng, 1, max(1, min(60000, (500 << 20) // (2 * batch * kv * dim))))
        window = rng.choice([0, 0, _log(rng, 1, max(1, length))])
        return dict(shape, batch=batch, length=length, window=window, sinks=rng.choice([0, 1, 4, 37]) if window else 0)
    if op == "append":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(2048, (400 << 20) // (4 * batch * (kv * group + 2 * kv) * dim))))
        return dict(shape, batch=batch, new=new, past=rng.choice([0, _log(rng, 1, 4000)]))
    batch = _log(rng, 1, 8)
    new = _log(rng, 1, 2048)
    past = rng.choice([0, _log(rng, 1, 3000)])
    new = max(1, min(new, (1 << 29) // (batch * kv * group * (new + past))))
    window = rng.choice([0, 0, _log(rng, 1, new + past)])
    return dict(shape, batch=batch, new=new, past=past, window=window, sinks=rng.choice([0, 1, 4, 37]) if window else 0, dtype="bfloat16")


def _spread(n, most, ragged):
    """n sizes of at most `most`, the first of them `most`: all alike, or spread over 0 .. most."""
    return [most if not ragged or i == 0 else (i * 7919 + 3 * most // 5) % (most + 1) for i in range(n)]


def _sizes(case):
    """Per sequence: (tokens in the cache before the pass, new tokens of the pass)."""
    batch, ragged = case["batch"], case.get("ragged", False)
    if case["op"] == "decode":
        lengths = [0 if ragged and i % 7 == 6 else n for i, n in enumerate(_spread(batch, case["length"], ragged))]  # some slots idle
        return [(max(0, n - 1), min(1, n)) for n in lengths]
    if case["op"] == "append" and case["new"] == 1:
        return [(case["past"] + 5 * i % 64, 1) for i in range(batch)]
    past = _spread(batch, case["past"], ragged)
    return list(zip(past[::-1], _spread(batch, case["new"], ragged)))


def _visible(case, p):
    """Keys that a query at position p sees."""
    w, s = case["window"], case["sinks"]
    return p + 1 if w == 0 or w > p else w + min(s, p + 1 - w)


def work(case):
    dim, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    if case["op"] == "pages":
        blocks = sum(-(-t // BLOCK) for t in _moved(case))
        return {"bytes": 2.0 * case["layers"] * blocks * 2 * kv * (BLOCK * dim + 4) + 24 * case["moves"], "flops": 0}
    heads, item = case["heads"], 4 if case["dtype"] == "float32" else 2
    sizes = _sizes(case)
    tokens = sum(n for _, n in sizes)
    table = 4.0 * sum(-(-(m + n) // page) for m, n in sizes)
    if case["op"] == "append":
        scales = sum(-(-(m + n) // BLOCK) - m // BLOCK for m, n in sizes if n) * kv * 2 * 4.0
        return {"bytes": tokens * ((heads + 2 * kv) * dim * 4 + heads * dim * item + 2 * kv * dim + dim * 4.0) + scales + table, "flops": tokens * dim * (heads + kv) * 3.0}
    pairs, read = 0, 0
    for m, n in sizes:
        pairs += sum(_visible(case, p) for p in range(m, m + n))
        if n:  # keys that some query of the sequence sees
            w, s = case["window"], case["sinks"]
            read += m + n if w == 0 else min(m + n, w + n - 1 + min(s, max(0, m - w + 1)))
    return {"bytes": read * kv * 2 * (dim + 4 / BLOCK) + tokens * heads * dim * 2 * item + table, "flops": 4.0 * heads * dim * pairs}


def _moved(case):
    """Tokens of each copied page."""
    return [1 + (37 * i) % case["page"] if case["partial"] else case["page"] for i in range(case["moves"])]


def _scale_of(amax):
    """The smallest power of two (at least 2^-120) of which amax is at most 448 times."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875)).clamp(min=-120))


def _codes(x):
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _pool(gen, layers, pages, kv, page, dim, outliers):
    """Codes and scales of a pool filled as a model's keys (a few channels several times the others) or values are."""
    x = torch.randn(layers, pages, kv, page // BLOCK, BLOCK, dim, generator=gen, device="cuda")
    x *= 0.5 + torch.rand(layers, pages, kv, page // BLOCK, 1, 1, generator=gen, device="cuda")
    if outliers:
        x[..., ::19] *= 5
    s = _scale_of(x.abs().amax((-1, -2)))
    return _codes(x.div_(s[..., None, None])).view(layers, pages, kv, page, dim), s


def _rope_table(positions, dim):
    f = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv, page, dim = case["kv_heads"], case["page"], case["head_dim"]
    s = {"case": case}
    if case["op"] == "pages":
        layers, pages = case["layers"], case["pages"]
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        s.update(src=order[:case["moves"]], dst=order[case["moves"]:2 * case["moves"]], tokens=_moved(case))
        parts = [_pool(gen, 1, pages, kv, page, dim, i % 2 == 0) for i in range(2 * layers)]
        s["k"], s["ks"] = (torch.cat([p[j].view(torch.uint8) if j == 0 else p[j] for p in parts[::2]]) for j in (0, 1))
        s["v"], s["vs"] = (torch.cat([p[j].view(torch.uint8) if j == 0 else p[j] for p in parts[1::2]]) for j in (0, 1))
        s["k"], s["v"] = s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)
    else:
        sizes = _sizes(case)
        heads, dtype = case["heads"], DTYPES[case["dtype"]]
        mapped = [-(-(m + n) // page) for m, n in sizes]
        pages, width = sum(mapped) + 3, max(1, max(mapped))
        s["k"], s["ks"] = _pool(gen, 1, pages, kv, page, dim, True)
        s["v"], s["vs"] = _pool(gen, 1, pages, kv, page, dim, False)
        first = torch.tensor([0] + mapped, device="cuda").cumsum(0)[:-1, None]
        at = torch.arange(width, device="cuda")[None, :]
        here = at < torch.tensor(mapped, device="cuda")[:, None]
        if case["op"] == "decode" and case["window"]:  # pages that hold no visible token are freed
            n = torch.tensor([m + k for m, k in sizes], device="cuda")[:, None]
            here &= ((at + 1) * page > n - case["window"]) | (at * page < case["sinks"])
        order = torch.randperm(pages, generator=gen, device="cuda")
        s["table"] = torch.where(here, order[(first + at).clamp(max=pages - 1)], -1).int()
        s["lengths"] = torch.tensor([m + n for m, n in sizes], dtype=torch.int32, device="cuda")
        s["starts"] = torch.tensor([m for m, _ in sizes], dtype=torch.int32, device="cuda")
        s["offsets"] = torch.tensor([0] + [n for _, n in sizes], device="cuda").cumsum(0).int()
        s["most_new"] = max(n for _, n in sizes)
        tokens = sum(n for _, n in sizes)
        if case["op"] == "append":
            s["qkv"] = torch.randn(tokens, (heads + 2 * kv) * dim, generator=gen, device="cuda")
            s["qkv"][:, ::37] *= 4
            s["rope"] = _rope_table(max(m + n for m, n in sizes), dim)
        else:
            rows = case["batch"] if case["op"] == "decode" else tokens
            s["q"] = torch.randn(rows, heads, dim, generator=gen, device="cuda").to(dtype)
    if own:  # the handle that a serving program keeps
        from jax4j_b200.kv8 import Kv8Cache
        s["cache"] = Kv8Cache.wrap(s["k"], s["v"], s["ks"], s["vs"])
    return s


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        cache = s["cache"]
        if op == "append":
            q = cache.append(s["qkv"], s["rope"], s["table"], s["starts"], heads=case["heads"],
                             offsets=None if case["new"] == 1 else s["offsets"], q_dtype=DTYPES[case["dtype"]])
            return {"q": q, "k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}
        if op == "decode":
            return cache.attention_decode(s["q"], s["table"], s["lengths"], window=case["window"], sinks=case["sinks"])
        if op == "prefill":
            return cache.attention_prefill(s["q"], s["offsets"], s["table"], s["lengths"], window=case["window"], sinks=case["sinks"])
        cache.copy_pages(s["src"], s["dst"], s["tokens"])
        return {"k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "pages": _plain_pages}[op](s)


def _plain_pages(s):
    case = s["case"]
    src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
    tokens = torch.tensor(s["tokens"], device="cuda")
    layers, pages, kv, page, dim = s["k"].shape
    moved = (torch.arange(page // BLOCK, device="cuda") * BLOCK < tokens[:, None])[None, :, None, :]  # [1, moves, 1, blocks]
    for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        c = codes.view(torch.uint8).view(layers, pages, kv, page // BLOCK, BLOCK * dim)
        c[:, dst] = torch.where(moved[..., None], c[:, src], c[:, dst]) if case["partial"] else c[:, src]
        scales[:, dst] = torch.where(moved, scales[:, src], scales[:, dst]) if case["partial"] else scales[:, src]
    return {"k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}


def _rotate(x, cs):
    """Adjacent pairs of x [tokens, heads, dim] by the angles whose (cos, sin) are cs [tokens, dim / 2, 2]."""
    x = x.unflatten(-1, (-1, 2))
    c, d = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack((x[..., 0] * c - x[..., 1] * d, x[..., 0] * d + x[..., 1] * c), -1).flatten(-2)


def _plain_append(s):
    case = s["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    tokens = s["qkv"].shape[0]
    seq = torch.searchsorted(s["offsets"][1:], torch.arange(tokens, dtype=torch.int32, device="cuda"), right=True)
    pos = s["starts"][seq] + torch.arange(tokens, device="cuda") - s["offsets"][seq]
    x = s["qkv"].view(tokens, heads + 2 * kv, dim)
    cs = s["rope"][pos]
    q = _rotate(x[:, :heads], cs).to(DTYPES[case["dtype"]])
    where = s["table"][seq, pos // page] * (page // BLOCK) + pos % page // BLOCK  # block of each token
    slot = pos % BLOCK
    old = s["starts"] % BLOCK  # tokens that the first block of each sequence holds already
    has = (s["offsets"][1:] > s["offsets"][:-1]) & (old > 0)
    head = s["table"].gather(1, (s["starts"] // page).clamp(max=s["table"].shape[1] - 1).long()[:, None])[:, 0] * (page // BLOCK) + s["starts"] % page // BLOCK
    for new, codes, scales in ((_rotate(x[:, heads:heads + kv], cs), s["k"], s["ks"]), (x[:, heads + kv:], s["v"], s["vs"])):
        c = codes[0].view(torch.uint8).view(-1, kv, page // BLOCK, BLOCK, dim)
        sc = scales[0].transpose(1, 2).flatten(0, 1)  # [blocks, kv], a copy
        amax = torch.zeros_like(sc).index_reduce_(0, where, new.abs().amax(-1), "amax")
        touched = torch.zeros(sc.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, where, True)
        kept = torch.zeros(sc.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, head[has].long(), True)
        fresh = _scale_of(amax)
        now = torch.where(touched[:, None], torch.where(kept[:, None], torch.maximum(fresh, sc), fresh), sc)
        hb, ho = head[has].long(), old[has]
        hp, hk = hb // (page // BLOCK), hb % (page // BLOCK)
        before = c[hp, :, hk].view(torch.float8_e4m3fn).float()  # [n, kv, 16, dim]
        again = _codes(before * (sc[hb] / now[hb])[:, :, None, None]).view(torch.uint8)
        mine = torch.arange(BLOCK, device="cuda")[None, None, :, None] < ho[:, None, None, None]
        c[hp, :, hk] = torch.where(mine, again, before.to(torch.float8_e4m3fn).view(torch.uint8))
        c[where // (page // BLOCK), :, where % (page // BLOCK), slot] = _codes(new / now[where][..., None]).view(torch.uint8)
        scales[0].copy_(now.view(-1, page // BLOCK, kv).transpose(1, 2))
    return {"q": q, "k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}


def _values(codes, scales, table):
    """[batch, kv_heads, width * page, dim] f32: the values of the pages that the table names (page 0 in the place of none)."""
    at = table.clamp(min=0)
    c = codes[0].view(torch.uint8)[at].view(torch.float8_e4m3fn).float().unflatten(3, (-1, BLOCK))  # [batch, width, kv, blocks, 16, dim]
    x = c * scales[0][at][..., None, None]
    return x.permute(0, 2, 1, 3, 4, 5).flatten(2, 4)


def _attend(q, s, at):
    """q [batch, kv_heads, group, n, dim] f32 at positions at [batch, n]."""
    case = s["case"]
    k, v = _values(s["k"], s["ks"], s["table"]), _values(s["v"], s["vs"], s["table"])
    j = torch.arange(k.shape[2], device="cuda")[None, None, :]
    p = at[..., None]
    seen = (j <= p) & (j < s["lengths"][:, None, None]) & (s["table"] >= 0).repeat_interleave(case["page"], 1)[:, None, :]
    if case["window"]:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    seen = seen[:, None, None]  # [batch, 1, 1, n, keys]
    x = torch.matmul(q.flatten(2, 3) * case["head_dim"] ** -0.5, k.transpose(-1, -2)).unflatten(2, q.shape[2:4])
    x.masked_fill_(~seen, -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=-3e38)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.flatten(2, 3), v).unflatten(2, q.shape[2:4])
    return o / total.clamp(min=1e-30)


def _plain_decode(s):
    case = s["case"]
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1)).unsqueeze(3)
    o = _attend(q, s, (s["lengths"] - 1)[:, None])
    return o.squeeze(3).flatten(1, 2).to(s["q"].dtype)


def _plain_prefill(s):
    case = s["case"]
    tokens = s["q"].shape[0]
    seq = torch.searchsorted(s["offsets"][1:], torch.arange(tokens, dtype=torch.int32, device="cuda"), right=True)
    i = torch.arange(tokens, device="cuda") - s["offsets"][seq]
    q = torch.zeros(case["batch"], s["most_new"], case["heads"], case["head_dim"], device="cuda")
    q[seq, i] = s["q"].float()
    o = _attend(q.permute(0, 2, 1, 3).unflatten(1, (case["kv_heads"], -1)), s, s["starts"][:, None] + torch.arange(s["most_new"], device="cuda")[None, :])
    return o.flatten(1, 2).permute(0, 2, 1, 3)[seq, i].to(s["q"].dtype)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)


def _exact_append(case, s):
    """Sequence by sequence and block by block of 16, in 64 bits."""
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if sum(-(-n // BLOCK) + 1 for _, n in _sizes(case)) > 3000:
        return None
    out = torch.zeros(s["qkv"].shape[0], heads, dim, dtype=torch.float64, device="cuda")
    codes = [s["k"][0].double(), s["v"][0].double()]
    scales = [s["ks"][0].double(), s["vs"][0].double()]
    table, row = s["table"].tolist(), 0
    for b, (past, n) in enumerate(_sizes(case)):
        x = s["qkv"][row:row + n].double().view(n, heads + 2 * kv, dim // 2, 2)
        turn = torch.view_as_complex(s["rope"][past:past + n].double())[:, None]
        turned = torch.view_as_real(torch.view_as_complex(x[:, :heads + kv].contiguous()) * turn).flatten(2)
        out[row:row + n] = turned[:, :heads]
        row += n
        done = 0
        while done < n:
            p = past + done
            take = min(n - done, BLOCK - p % BLOCK)
            pg, blk, slot = table[b][p // page], p % page // BLOCK, p % BLOCK
            for i, new in enumerate((turned[done:done + take, heads:], x[done:done + take, heads + kv:].flatten(2))):
                most = new.abs().amax((0, 2))
                e = torch.ceil(torch.log2(most / 448)).clamp(min=-120)
                e = torch.where(most > 448 * 2.0 ** e, e + 1, torch.where(most <= 448 * 2.0 ** (e - 1), e - 1, e))
                now = 2.0 ** e
                lo = blk * BLOCK
                if slot:
                    now = torch.maximum(now, scales[i][pg, :, blk])
                    kept = codes[i][pg, :, lo:lo + slot] * (scales[i][pg, :, blk] / now)[:, None, None]
                    codes[i][pg, :, lo:lo + slot] = kept.to(torch.float8_e4m3fn).double()
                scales[i][pg, :, blk] = now
                codes[i][pg, :, lo + slot:lo + slot + take] = (new.transpose(0, 1) / now[:, None, None]).to(torch.float8_e4m3fn).double()
            done += take
    return {"q": out, "k": codes[0][None], "k_scale": scales[0][None], "v": codes[1][None], "v_scale": scales[1][None]}


def _exact_attention(case, s):
    """Query tile by query tile, in 64 bits, over the keys gathered in order."""
    kv, page, dim = case["kv_heads"], case["page"], case["head_dim"]
    group = case["heads"] // kv
    decode = case["op"] == "decode"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    table, row = s["table"].tolist(), 0
    for b, (past, n) in enumerate(_sizes(case)):
        if n:
            keys = torch.arange(past + n, device="cuda")
            at = torch.tensor(table[b], device="cuda")[keys // page]
            there = at >= 0
            keys, at = keys[there], at[there]
            blk, slot = keys % page // BLOCK, keys % page
            k, v = (c[0].view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn).double() * sc[0][at, :, blk].double()[..., None] for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for lo in range(0, n, 512):
                m = min(512, n - lo)
                q = s["q"][row + lo:row + lo + m].double().view(m, kv, group, dim)
                x = torch.einsum("mhgd,khd->hgmk", q, k) / math.sqrt(dim)
                p = torch.arange(past + lo, past + lo + m, device="cuda")[:, None]
                hide = keys[None] > p
                if case["window"]:
                    hide |= (keys[None] <= p - case["window"]) & (keys[None] >= case["sinks"])
                w = torch.softmax(x.masked_fill(hide, -math.inf), -1).nan_to_num(0.0)
                out[row + lo:row + lo + m] = torch.einsum("hgmk,khd->mhgd", w, v).reshape(m, kv * group, dim)
        row += 1 if decode else n
    return out
