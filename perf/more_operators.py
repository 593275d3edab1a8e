"""The operators on caches of pages, as they are timed: each in its plain form (elementary torch operations in 32 bits,
64 where a selection hangs on it) and, where `own` is true, through the public binding, leap_amd.attention.

A case is a dict of plain values:
  kind       "step": PagedAttention.step_async, one new token of every sequence over its pages
             "sparse": PagedAttention.step_sparse_async, the same over the pages that a score of their keys picks
             "fork": PagedAttention.fork_async and reserve_async: sequences continue from others' pages, which they
                 share, and get a page of their own for the row that each will write (a copy where it is shared)
             "compact": PagedAttention.fork_async, compact_async and reserve_async: sequences end, the pages behind
                 them move into their place, and others begin
             "beam": PagedAttention.beam_select_async, the best beams of each group over all beams and the vocabulary
  heads, kv_heads, head_dim, theta   the model's head shape and RoPE base
  layers     layers the handle holds; a step runs each of them once
  page_rows  rows of a page
  q8         a cache of int8 values with a scale per row and KV head (else fp32)
  batch, ctx, shortest, len_seed     sequences; rows of each with its new token (shortest..ctx, the first has ctx); the
             seed they are drawn with
  keep       "sparse": pages that a query attends to at most
  sources    "fork": sequences that the others continue from
  groups, beams, vocab               "beam"
"""
import math
import random

import torch

own = False

DEV = "cuda"

# (q heads, KV heads, head_dim, RoPE base, layers of the model)
TINY = (32, 4, 64, 10000.0, 22)
L3_8B = (32, 8, 128, 500000.0, 32)
L2_7B = (32, 32, 128, 10000.0, 32)
L3_70B = (64, 8, 128, 500000.0, 80)
L31_405B = (128, 8, 128, 500000.0, 126)


def _case(kind, model, layers, batch, ctx, shortest=None, len_seed=0, page_rows=16, q8=False, keep=0, sources=0, name=None):
    c = {"kind": kind, "heads": model[0], "kv_heads": model[1], "head_dim": model[2], "theta": model[3],
         "layers": layers, "page_rows": page_rows, "q8": q8, "batch": batch, "ctx": ctx,
         "shortest": ctx if shortest is None else shortest, "len_seed": len_seed}
    if kind == "sparse":
        c["keep"] = keep
    if kind == "fork":
        c["sources"] = sources
    return {"name": name, **c} if name else c


def _beam(groups, beams, vocab, name=None):
    c = {"kind": "beam", "groups": groups, "beams": beams, "vocab": vocab}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a short conversation with a small model: a launch is all there is
        _case("step", TINY, 22, 1, 256, name="step-tinyllama-ctx256"),
        # the benchmark's headline with its cache in pages
        _case("step", L3_8B, 16, 1, 4096, name="step-llama3-8b-ctx4096"),
        # a server's batch on a large model's stage, conversations of all lengths
        _case("step", L3_70B, 2, 16, 7300, shortest=411, len_seed=5, page_rows=32, name="step16-llama3-70b-ragged7300"),
        # a larger batch on an 8-bit cache
        _case("step", L3_8B, 4, 32, 8192, shortest=300, len_seed=7, q8=True, name="step32-llama3-8b-q8-ragged8192"),
        # a long document in one request, decoding with a thirty-second of its pages
        _case("sparse", L3_8B, 4, 1, 65536, page_rows=32, keep=64, name="sparse-llama3-8b-ctx65536"),
        # a batch of long conversations on an 8-bit cache
        _case("sparse", L3_8B, 2, 16, 16384, shortest=1999, len_seed=3, page_rows=32, q8=True, keep=48,
              name="sparse16-llama3-8b-q8-ragged16384"),
        # four beams of a small model go on from two of them
        _case("fork", TINY, 22, 4, 257, sources=2, name="fork4-tinyllama-ctx257"),
        # a long prompt answered in sixty-four samples: shared pages, a last one each
        _case("fork", L3_8B, 8, 64, 3001, shortest=2900, len_seed=9, sources=8, name="fork64-llama3-8b-ragged3001"),
        # a small model's pool with holes, made dense
        _case("compact", TINY, 22, 3, 500, shortest=33, len_seed=2, name="compact3-tinyllama-ragged500"),
        # a server's pool after half of its conversations ended
        _case("compact", L3_8B, 4, 8, 2011, shortest=100, len_seed=4, page_rows=32, name="compact8-llama3-8b-ragged2011"),
        # beams of one request over a small vocabulary
        _beam(1, 4, 32000, name="beam1x4-32000"),
        # a batch of requests with eight beams over a large one
        _beam(24, 8, 128256, name="beam24x8-128256"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "sparse", "sparse", "fork", "compact", "beam", "beam"])
    if kind == "beam":
        groups, beams, vocab = _log_int(rng, 1, 64), rng.randint(1, 16), _log_int(rng, 500, 131072)
        return _beam(min(groups, max(1, 24 * 8 * 128256 // (beams * vocab))), beams, vocab)
    model = rng.choice([TINY, L3_8B, L2_7B, L3_70B, L31_405B])
    q8 = rng.random() < 0.5
    page_rows = rng.choice([16, 16, 32, 64, 128])
    seed = rng.randrange(1 << 16)
    short = lambda ctx: ctx if rng.random() < 0.3 else max(1, int(ctx * rng.uniform(0.05, 0.9)))  # noqa: E731
    if kind in ("step", "sparse"):
        ctx = _log_int(rng, 16 if kind == "step" else 256, 65536 if model is not L2_7B else 8192)
        batch = 1 if rng.random() < 0.4 else min(_log_int(rng, 2, 64), max(2, (1 << 18) // ctx))
        c = _case(kind, model, 1, batch, ctx, short(ctx), seed, page_rows, q8, keep=rng.choice([1, 4, 16, 37, 64, 128]))
        w = work(c)
        # as many of the model's layers as keep a pass small
        c["layers"] = max(1, min(model[4], 16, int(2e8 / w["bytes"])))
        while c["batch"] > 1 and (_pool_bytes(c) > 1.6e10 or work(c)["bytes"] > 1.3e9 or work(c)["flops"] > 7e9):
            c["batch"] -= 1
        return c
    batch, ctx = _log_int(rng, 1, 64 if kind == "fork" else 12), _log_int(rng, 1, 4096)
    c = _case(kind, model, 1, batch, ctx, short(ctx), seed, page_rows, q8 and kind == "fork", sources=rng.randint(1, batch))
    most = {"fork": 4e8, "compact": 6e8}[kind]
    c["layers"] = max(1, min(model[4], 8, int(most / work(c)["bytes"])))
    while c["batch"] > 1 and work(c)["bytes"] > most:
        c["batch"] -= 1
    if kind == "fork":
        c["sources"] = min(c["sources"], c["batch"])
    return c


def sizes(c):
    """Rows of each sequence, the new one with them."""
    r = random.Random(c["len_seed"])
    return [c["ctx"]] + [r.randint(c["shortest"], c["ctx"]) for _ in range(c["batch"] - 1)]


def _pages_of(rows, c):
    return -(-rows // c["page_rows"])


def _parents(c, seed):
    """"fork": which source each sequence continues from."""
    r = random.Random(seed * 7919 + 17)
    return [r.randrange(c["sources"]) for _ in range(c["batch"])]


def _pool(c):
    """Pages of the pool."""
    n = [_pages_of(x, c) for x in sizes(c)]
    if c["kind"] == "fork":
        return sum(n[:c["sources"]]) + 2 * c["batch"] + 3
    if c["kind"] == "compact":
        return 2 * sum(n) + 5
    return sum(n) + _pages_of(c["ctx"], c) + 3  # (as many again as the longest has, for another tenant)


def _row_bytes(c):
    return c["kv_heads"] * (c["head_dim"] + 4 if c["q8"] else 4 * c["head_dim"])  # of K or of V


def _pool_bytes(c):
    return 2 * _pool(c) * c["page_rows"] * _row_bytes(c) * c["layers"]


def _held(c):
    """Sequences that the handle has."""
    return {"fork": c["batch"] + c.get("sources", 0), "compact": 2 * c["batch"]}.get(c["kind"], c["batch"] + 1)


def work(c):
    if c["kind"] == "beam":
        n = c["groups"] * c["beams"]
        return {"bytes": 4 * n * c["vocab"] + 16 * n, "flops": 4 * n * c["vocab"]}
    H, G, hd, R, L = c["heads"], c["kv_heads"], c["head_dim"], c["page_rows"], c["layers"]
    row = 2 * _row_bytes(c)
    rows, b, f = sizes(c), 0, 0
    if c["kind"] in ("step", "sparse"):
        for n in rows:
            seen = n - 1
            if c["kind"] == "sparse":
                full = (n - 1) // R  # pages with a score
                seen = min(seen, (c["keep"] - 1) * R + (n - 1) % R)
                if _pages_of(n, c) > c["keep"]:
                    b += full * 8 * G * hd
                    f += 3 * full * H * hd
            b += seen * row + 8 * H * hd + 8 * G * hd + row + 4 * _pages_of(n, c)
            f += 4 * (seen + 1) * H * hd
        return {"bytes": b * L, "flops": f * L}
    pages = [_pages_of(n, c) for n in rows]
    if c["kind"] == "fork":
        src = [pages[p] for p in _parents(c, 0)]
        return {"bytes": 8 * sum(src) + c["batch"] * 2 * R * row * L, "flops": 4 * sum(src)}
    return {"bytes": 16 * sum(pages) + sum(pages) * 2 * R * row * L, "flops": 4 * sum(pages)}


# ---- where the pages are -----------------------------------------------------

def _rounds(c):
    """The reservations that fill the tables, [(from, to) of every sequence]: the sequences grow in turn, as
    conversations do, with another tenant among them."""
    n = sizes(c)
    if c["kind"] == "fork":
        return [([0] * _held(c), [0] * c["batch"] + n[:c["sources"]])]
    if c["kind"] == "compact":
        return [([0] * _held(c), n + [0] * c["batch"]), (n + [0] * c["batch"], n + n)]
    ends, out, before = n + [c["ctx"]], [], [0] * (len(n) + 1)
    for r in range(1, 13):
        to = [max(a, e * r // 12) for a, e in zip(before, ends)]
        out.append((before, to))
        before = to
    return out


def _tables(c):
    """[sequences][pages of the longest]: page numbers (-1: none), and the next free one.  Pages are given in ascending
    order, sequence after sequence."""
    width = _width(c)
    t, free = [[-1] * width for _ in range(_held(c))], 0
    for _, to in _rounds(c):
        for row, rows in zip(t, to):
            for j in range(_pages_of(rows, c)):
                if row[j] < 0:
                    row[j], free = free, free + 1
    return t, free


def _seq_len(c):
    return max(128, 1 << (c["ctx"] - 1).bit_length())


def _width(c):
    return _pages_of(_seq_len(c), c)


# ---- inputs --------------------------------------------------------------------

def _gen(seed, *what):
    s = seed & 0xFFFFFFFF
    for w in what:
        s = (s * 1000003 + w + 12345) & 0x7FFFFFFFFFFF
    return torch.Generator(device=DEV).manual_seed(s)


def _tokens(c, seed):
    """q, k and v of the new tokens, [layers][batch][...]; queries of twice the keys' spread give scores with the few
    heavy rows that trained attention has."""
    g = _gen(seed, 2)
    B, L, hd = c["batch"], c["layers"], c["head_dim"]
    q = torch.randn(L, B, c["heads"] * hd, device=DEV, generator=g) * 2.0
    k = torch.randn(L, B, c["kv_heads"] * hd, device=DEV, generator=g)
    v = torch.randn(L, B, c["kv_heads"] * hd, device=DEV, generator=g)
    return q, k, v


def _logits(c, seed):
    """Logits with a few likely tokens, and the beams' scores so far."""
    g = _gen(seed, 5)
    n = c["groups"] * c["beams"]
    x = torch.randn(n, c["vocab"], device=DEV, generator=g) * 2.5
    likely = torch.randint(0, c["vocab"], (n, 8), device=DEV, generator=g)
    x.scatter_add_(1, likely, torch.rand(n, 8, device=DEV, generator=g) * 12.0)
    scores = -20.0 * torch.rand(n, device=DEV, generator=g)
    return x, scores


def _shapes(c):
    """The pool's arrays: name, shape, dtype.  A KV head's rows of a page lie together; 8-bit values in V of 16 rows
    dimension by dimension."""
    L, P, G, R, hd = c["layers"], _pool(c), c["kv_heads"], c["page_rows"], c["head_dim"]
    if not c["q8"]:
        s = [("k", (L, P, G, R, hd), torch.float32), ("v", (L, P, G, R, hd), torch.float32)]
    else:
        s = [("k", (L, P, G, R, hd), torch.int8), ("v", (L, P, G, R // 16, hd, 16), torch.int8),
             ("ks", (L, P, G, R), torch.float32), ("vs", (L, P, G, R), torch.float32)]
    if c["kind"] == "sparse":
        s.append(("bounds", (L, P, G, 2, hd), torch.float32))
    return s


class _DeviceArray:
    """An array in device memory of a handle, for torch.as_tensor."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


def _arrays(c, h):
    """The pool's arrays, of a handle or (h None) of the plain form."""
    out = {}
    view = h.view(0) if h else None
    for name, shape, dtype in _shapes(c):
        if h:
            out[name] = torch.as_tensor(_DeviceArray(h, view[name], shape, "|i1" if dtype == torch.int8 else "<f4"), device=DEV)
        else:
            out[name] = torch.empty(shape, dtype=dtype, device=DEV)
    return out


def _fill(c, seed, pool):
    """Rows of a pool: unit keys, as after RoPE, and values (8 bits: of a normal spread whose largest is near 127, and
    scales of such rows), and the least and largest of each page's keys."""
    for i, name in enumerate(("k", "v")):
        g, t = _gen(seed, 3, i), pool[name]
        if c["q8"]:
            for x in t.flatten(0, 1).split(64):
                x.copy_(torch.randn(x.shape, device=DEV, generator=g).mul_(45.0).round_().clamp_(-127, 127))
            pool[name + "s"].uniform_(2.0 / 127, 3.0 / 127, generator=g)
        else:
            t.normal_(generator=g)
    if "bounds" in pool:
        for l in range(c["layers"]):
            for at in range(0, _pool(c), 256):
                x = _keys(c, pool, l)[at:at + 256]
                pool["bounds"][l, at:at + 256] = torch.stack((x.amin(dim=-2), x.amax(dim=-2)), dim=-2)


class _Values:
    """Keys or values of a layer's pages, as the fp32 numbers they stand for, read where they are indexed."""

    def __init__(self, values, scales, blocks):
        self.values, self.scales, self.blocks = values, scales, blocks

    def __getitem__(self, at):
        x = self.values[at]
        if self.scales is None:
            return x
        if self.blocks:  # [...][rows / 16][head_dim][16]
            x = x.transpose(-1, -2).flatten(-3, -2)
        return x.float() * self.scales[at][..., None]


def _keys(c, pool, l):
    return _Values(pool["k"][l], pool["ks"][l] if c["q8"] else None, False)


def _vals(c, pool, l):
    return _Values(pool["v"][l], pool["vs"][l] if c["q8"] else None, True)


def _rope_table(c):
    """cos and sin of the rotary angles, [seq_len][head_dim / 2].  The engine's table rounds frequencies and angles
    to fp32, which is part of its definition: base 500000 is a constant of its build, whose powers its compiler
    forms as exp(-i log(base)) with the exponent in fp32."""
    hd, base = c["head_dim"], c["theta"]
    i = torch.arange(0, hd, 2, dtype=torch.float32, device=DEV) / hd
    if base == 500000.0:
        freq = torch.exp((-i * torch.tensor(math.log(base), dtype=torch.float32, device=DEV)).double()).float()
    else:
        freq = (1.0 / torch.pow(torch.tensor(base, dtype=torch.float64, device=DEV), i.double())).float()
    a = (torch.arange(_seq_len(c), dtype=torch.float32, device=DEV)[:, None] * freq).double()
    return torch.cos(a).float(), torch.sin(a).float()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(c, seed):
    """The pool filled and the tables laid as a program holds them when the tokens come (in a handle, for the framework's
    operators), and the call's buffers."""
    st = {"c": c}
    if c["kind"] == "beam":
        st["logits"], st["scores"] = _logits(c, seed)
        n = c["groups"] * c["beams"]
        st["parent"], st["token"], st["best"] = _i32([0] * n), _i32([0] * n), torch.empty(n, device=DEV)
        if own:
            from leap_amd.attention import PagedAttention
            st["h"] = PagedAttention(8, 4, 64, 16, n_pages=1, max_batch=n)
        torch.cuda.synchronize()
        return st
    tables, free = _tables(c)
    h = None
    if own:
        from leap_amd.attention import PagedAttention
        h = PagedAttention(c["heads"], c["kv_heads"], c["head_dim"], _seq_len(c), n_pages=_pool(c), page_rows=c["page_rows"],
                           n_layers=c["layers"], rope_theta=c["theta"], max_batch=_held(c), cache="q8" if c["q8"] else "f32",
                           bounds=c["kind"] == "sparse")
        for begin, end in _rounds(c):
            h.reserve(begin, end)
        at = h.view(0)
        st["table"] = torch.as_tensor(_DeviceArray(h, at["table"], (_held(c), _width(c)), "<i4"), device=DEV)
        st["refs"] = torch.as_tensor(_DeviceArray(h, at["refs"], (_pool(c),), "<i4"), device=DEV)
    else:
        st["table"] = _i32(tables)
        st["refs"] = (torch.arange(_pool(c), device=DEV) < free).int()
    st["h"], st["pool"] = h, _arrays(c, h)
    _fill(c, seed, st["pool"])
    n, B = sizes(c), c["batch"]
    if c["kind"] in ("step", "sparse"):
        st["rope"] = _rope_table(c)
        st["qkv"] = q, _, _ = _tokens(c, seed)
        st["out"] = torch.empty_like(q)
        st["pos"], st["max_pos"], st["rows"] = _i32([x - 1 for x in n]), max(n) - 1, sum(n)
        # where the new rows are
        st["new_page"] = torch.tensor([tables[i][(x - 1) // c["page_rows"]] for i, x in enumerate(n)], device=DEV)
        st["new_row"] = torch.tensor([(x - 1) % c["page_rows"] for x in n], device=DEV)
        if c["kind"] == "sparse":
            st["picked"] = _i32([[[[0] * c["keep"]] * c["kv_heads"]] * B] * c["layers"])
    elif c["kind"] == "fork":
        p = _parents(c, seed)
        st["from"], st["parent"] = [n[i] for i in p], _i32([B + i for i in p])
        # each goes on behind its source's last row but one, so that the row it will write lies in a shared page
        st["keep"] = _i32([max(1, x - 1) for x in st["from"]])
        st["to"] = _i32([max(1, x - 1) + 1 for x in st["from"]])
        st["status"] = _i32([0] * B)
        st["last"] = torch.tensor([max(1, x - 1) // c["page_rows"] for x in st["from"]], device=DEV)
    else:
        st["cut"], st["none"], st["rows"] = _i32([0] * B), _i32([0] * B), _i32(n)
        st["swap"] = _i32([B + i for i in range(B)] + list(range(B)))
        st["both"] = _i32(n + n)
        st["status"] = _i32([0] * B)
        st["count"] = _i32([0])
    torch.cuda.synchronize()
    return st


# ---- one pass -------------------------------------------------------------------

def _new_rows(st):
    """The rows of the new tokens as the cache holds them after the call, [batch][layers][kv_heads][head_dim]."""
    c, pool = st["c"], st["pool"]
    page, row = st["new_page"], st["new_row"]
    if not c["q8"]:
        return [pool[x][:, page, :, row] for x in ("k", "v")]
    k = pool["k"][:, page, :, row].float() * pool["ks"][:, page, :, row][..., None]
    v = pool["v"][:, page, :, row // 16, :, row % 16].float() * pool["vs"][:, page, :, row][..., None]
    return [k, v]


def _forked(st):
    """What a fork leaves: the table, and the pages that the sequences will write, of every layer."""
    c, pool = st["c"], st["pool"]
    table = st["table"]
    page = table[:c["batch"]].long().gather(1, st["last"][:, None])[:, 0]
    if not c["q8"]:
        return [table, st["refs"], pool["k"][:, page], pool["v"][:, page]]
    at = (slice(None), page)
    return [table, st["refs"]] + [_Values(pool[x], pool[x + "s"], x == "v")[at] for x in ("k", "v")]


def _run_own(st):
    c, h = st["c"], st["h"]
    kind = c["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "beam":
        h.beam_select_async(c["groups"], c["beams"], c["vocab"], st["logits"].data_ptr(), c["vocab"], st["scores"].data_ptr(),
                            st["parent"].data_ptr(), st["token"].data_ptr(), st["best"].data_ptr(), stream)
        return [st["parent"], st["token"], st["best"]]
    B = c["batch"]
    if kind == "fork":
        h.fork_async(B, st["parent"].data_ptr(), st["keep"].data_ptr(), stream)
        h.reserve_async(B, st["keep"].data_ptr(), st["to"].data_ptr(), st["status"].data_ptr(), stream)
        return _forked(st)
    if kind == "compact":
        h.fork_async(B, 0, st["cut"].data_ptr(), stream)
        h.compact_async(st["count"].data_ptr(), stream)
        h.reserve_async(B, st["none"].data_ptr(), st["rows"].data_ptr(), st["status"].data_ptr(), stream)
        h.fork_async(2 * B, st["swap"].data_ptr(), st["both"].data_ptr(), stream)
        return [st["table"], st["refs"], st["count"], st["pool"]["k"], st["pool"]["v"]]
    q, k, v = st["qkv"]
    out, pos = st["out"], st["pos"].data_ptr()
    for l in range(c["layers"]):
        at = (q[l].data_ptr(), k[l].data_ptr(), v[l].data_ptr(), out[l].data_ptr())
        if kind == "step":
            h.step_async(l, B, pos, st["max_pos"], *at, stream, total_rows=st["rows"])
        else:
            h.step_sparse_async(l, B, pos, st["max_pos"], c["keep"], *at, st["picked"][l].data_ptr(), stream)
    return [out] + ([st["picked"]] if kind == "sparse" else []) + _new_rows(st)


def _rotate(x, cs, sn):
    """Interleaved pairs of each head; x [batch][heads][head_dim], cs and sn [batch][head_dim / 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    cs, sn = cs[:, None], sn[:, None]
    return torch.stack((a * cs - b * sn, b * cs + a * sn), dim=-1).flatten(-2)


def _quantize(x):
    """int8 values and one scale per head row."""
    a = x.abs().amax(dim=-1).clamp_min(2.0 ** -100)
    t = torch.full_like(a, 127.0)
    return torch.round(x * (t / a)[..., None]).to(torch.int8), a / t


def _attend(q, keys, vals, see):
    """q [...][heads of a KV head][head_dim] over keys and vals [...][rows][head_dim] where see [...][rows]."""
    s = torch.matmul(q, keys.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(q.shape[-1]))
    s = s.masked_fill_(~see[..., None, :], -math.inf)
    p = torch.exp_(s.sub_(s.amax(dim=-1, keepdim=True)))
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, vals.contiguous()) / total


def _step_plain(st):
    c, pool = st["c"], st["pool"]
    B, H, G, hd, R = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page_rows"]
    pos = st["pos"].long()
    cs, sn = st["rope"][0][pos], st["rope"][1][pos]
    width = st["max_pos"] // R + 1
    table = st["table"][:B, :width].long().clamp_min(0)
    page, row = st["new_page"], st["new_row"]
    for l in range(c["layers"]):
        q = _rotate(st["qkv"][0][l].unflatten(-1, (H, hd)), cs, sn)
        k = _rotate(st["qkv"][1][l].unflatten(-1, (G, hd)), cs, sn)
        v = st["qkv"][2][l].unflatten(-1, (G, hd))
        if c["q8"]:
            pool["k"][l][page, :, row], pool["ks"][l][page, :, row] = _quantize(k)
            pool["v"][l][page, :, row // 16, :, row % 16], pool["vs"][l][page, :, row] = _quantize(v)
        else:
            pool["k"][l][page, :, row], pool["v"][l][page, :, row] = k, v
        q = q.unflatten(1, (G, H // G))
        if c["kind"] == "step":
            keys, vals = (x[table].transpose(1, 2).flatten(2, 3) for x in (_keys(c, pool, l), _vals(c, pool, l)))
            see = (torch.arange(width * R, device=DEV) <= pos[:, None])[:, None].expand(B, G, width * R)
        else:
            # a page's score is the most that its keys' bounds allow, summed over the KV head's queries; the page of the
            # new row is always attended to, and of equal scores the earlier page is taken
            pages = (pos // R)[:, None, None]  # of the new row
            ends = _keys(c, pool, l)[page]  # (a page that the row completes has new bounds)
            full = (row == R - 1)[:, None, None, None]
            bounds = torch.stack((ends.amin(dim=-2), ends.amax(dim=-2)), dim=-2)
            pool["bounds"][l][page] = torch.where(full, bounds, pool["bounds"][l][page])
            score = torch.empty(B, G, width, dtype=torch.float64, device=DEV)
            for b in range(B):
                lo, hi = pool["bounds"][l][table[b]].double().transpose(0, 1).unbind(dim=2)  # [G][pages][hd]
                score[b] = sum(torch.maximum(x[:, None] * lo, x[:, None] * hi).sum(dim=-1) for x in q[b].double().unbind(dim=1))
            at = torch.arange(width, device=DEV)
            score.masked_fill_(at > pages, -math.inf)
            score.masked_fill_(at == pages, math.inf)
            best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
            some = best <= pages
            best = torch.sort(torch.where(some, best, width), dim=-1).values
            some = best < width
            pick = torch.where(some, best, 0)
            ids = table[:, None].expand(B, G, width).gather(2, pick)
            heads = torch.arange(G, device=DEV)[:, None]
            keys, vals = (x[ids, heads].flatten(2, 3) for x in (_keys(c, pool, l), _vals(c, pool, l)))
            rows = pick[..., None] * R + torch.arange(R, device=DEV)
            see = (some[..., None] & (rows <= pos[:, None, None, None])).flatten(2, 3)
            st["picked"][l].fill_(-1)
            st["picked"][l][..., :best.shape[-1]] = torch.where(some, best, -1).int()
        st["out"][l] = _attend(q, keys, vals, see).reshape(B, H * hd)
    return [st["out"]] + ([st["picked"]] if c["kind"] == "sparse" else []) + _new_rows(st)


def _fork_plain(st, n, parent, rows):
    """Sequences 0..n-1 take the pages of their parents' first rows."""
    c, table, refs = st["c"], st["table"], st["refs"]
    new = table[parent.long()].clone()
    new[torch.arange(new.shape[1], device=DEV) >= (rows[:, None] + c["page_rows"] - 1) // c["page_rows"]] = -1
    for t, by in ((new, 1), (table[:n], -1)):
        refs += by * torch.bincount(t[t >= 0].long(), minlength=refs.numel()).int()
    table[:n] = new


def _reserve_plain(st, n, begin, end):
    """Every page of rows [begin, end) of sequences 0..n-1 there, and its own: missing ones are the lowest free pages,
    shared ones copies."""
    c, table, refs, pool = st["c"], st["table"], st["refs"], st["pool"]
    R = c["page_rows"]
    at = torch.arange(table.shape[1], device=DEV)
    wanted = (at >= (begin // R)[:, None]) & (at * R < end[:, None])
    old = table[:n]
    # of the sequences that share a page and all will write it, the last keeps it
    ask = wanted & (old >= 0)
    i, j = ask.nonzero(as_tuple=True)
    page = old[i, j].long()
    asked = torch.bincount(page, minlength=refs.numel())
    last = torch.full((refs.numel(),), -1, device=DEV).scatter_reduce_(0, page, i, "amax")
    keeps = (refs[page] == 1) | ((asked[page] == refs[page]) & (last[page] == i))
    copy = torch.zeros_like(ask)
    copy[i[~keeps], j[~keeps]] = True
    i, j = (copy | (wanted & (old < 0))).nonzero(as_tuple=True)
    free = (refs == 0).nonzero()[:i.numel(), 0]
    source = old[i, j].long()
    has = source >= 0
    for x in pool.values():
        x[:, free[has]] = x[:, source[has]]
    refs -= torch.bincount(source[has], minlength=refs.numel()).int()
    refs[free] = 1
    table[i, j] = free.int()


def _compact_plain(st):
    """The pages in use move down until none is free below one; their order stays."""
    table, refs, pool = st["table"], st["refs"], st["pool"]
    used = refs > 0
    n = used.sum()
    at = torch.arange(refs.numel(), device=DEV)
    to, source = (~used & (at < n)).nonzero()[:, 0], (used & (at >= n)).nonzero()[:, 0]
    for x in pool.values():
        x[:, to] = x[:, source]
    refs[to] = refs[source]
    refs[source] = 0
    where = at.clone()
    where[source] = to
    table.copy_(torch.where(table >= 0, where[table.long().clamp_min(0)].int(), table))
    st["count"].copy_(n.int()[None])


def _beam_plain(st):
    c = st["c"]
    x = st["logits"]
    m = x.amax(dim=-1, keepdim=True)
    lse = m.double() + torch.log(torch.exp(x - m).double().sum(dim=-1, keepdim=True))
    total = (x.double() - lse + st["scores"].double()[:, None]).reshape(c["groups"], -1)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    best, at = best[:, :c["beams"]], at[:, :c["beams"]]
    beam = at // c["vocab"] + torch.arange(c["groups"], device=DEV)[:, None] * c["beams"]
    st["parent"].copy_(beam.reshape(-1))
    st["token"].copy_((at % c["vocab"]).reshape(-1))
    st["best"].copy_(best.reshape(-1))
    return [st["parent"], st["token"], st["best"]]


def _run_plain(st):
    c = st["c"]
    if c["kind"] == "beam":
        return _beam_plain(st)
    if c["kind"] in ("step", "sparse"):
        return _step_plain(st)
    B = c["batch"]
    if c["kind"] == "fork":
        _fork_plain(st, B, st["parent"], st["keep"])
        _reserve_plain(st, B, st["keep"], st["to"])
        return _forked(st)
    _fork_plain(st, B, torch.arange(B, device=DEV), st["cut"])
    _compact_plain(st)
    _reserve_plain(st, B, st["none"], st["rows"])
    _fork_plain(st, 2 * B, st["swap"], st["both"])
    return [st["table"], st["refs"], st["count"], st["pool"]["k"], st["pool"]["v"]]


def run(st):
    return _run_own(st) if own else _run_plain(st)


# ---- the same in 64 bits ----------------------------------------------------------

def _exact_beam(c, seed):
    x, scores = _logits(c, seed)
    parent, token, best = [], [], []
    for i in range(c["groups"]):
        here = slice(i * c["beams"], (i + 1) * c["beams"])
        total = torch.log_softmax(x[here].double(), dim=-1) + scores[here].double()[:, None]
        flat = total.reshape(-1)
        # (the largest few suffice; ties at the border keep the earlier place)
        least = torch.topk(flat, min(c["beams"], flat.numel())).values[-1]
        at = (flat >= least).nonzero()[:, 0].tolist()
        at.sort(key=lambda p: (-float(flat[p]), p))
        for p in at[:c["beams"]]:
            parent.append(i * c["beams"] + p // c["vocab"])
            token.append(p % c["vocab"])
            best.append(float(flat[p]))
    return [_i32(parent), _i32(token), torch.tensor(best, dtype=torch.float64, device=DEV)]


def _exact_tables(c, seed):
    """The tables and references after a pass of "fork" or "compact", and the page that each page's contents are of."""
    table, used = _tables(c)
    n, B = sizes(c), c["batch"]
    refs = [1 if p < used else 0 for p in range(_pool(c))]
    holds = list(range(_pool(c)))

    def drop(p):
        refs[p] -= 1

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    def fork(parents, rows):
        new = [[p if j < _pages_of(r, c) else -1 for j, p in enumerate(table[a])] for a, r in zip(parents, rows)]
        for t in new:
            for p in t:
                if p >= 0:
                    refs[p] += 1
        for i, t in enumerate(new):
            for p in table[i]:
                if p >= 0:
                    drop(p)
            table[i] = t

    def reserve(begin, end):
        for i, (a, e) in enumerate(zip(begin, end)):
            for j in range(a // c["page_rows"], _pages_of(e, c)):
                p = table[i][j]
                if p < 0:
                    table[i][j] = take()
                elif refs[p] > 1:
                    new = take()
                    drop(p)
                    holds[new], table[i][j] = holds[p], new

    if c["kind"] == "fork":
        p = _parents(c, seed)
        keep = [max(1, n[i] - 1) for i in p]
        fork([B + i for i in p], keep)
        reserve(keep, [x + 1 for x in keep])
        return table, refs, holds, [table[i][x // c["page_rows"]] for i, x in enumerate(keep)]
    fork(list(range(B)), [0] * B)
    count = sum(r > 0 for r in refs)
    to = [p for p in range(count) if refs[p] == 0]
    source = [p for p in range(count, len(refs)) if refs[p] > 0]
    move = dict(zip(source, to))
    for s, t in move.items():
        refs[t], refs[s], holds[t] = refs[s], 0, holds[s]
    table[:] = [[move.get(p, p) for p in t] for t in table]
    reserve([0] * B, n)
    fork([B + i for i in range(B)] + list(range(B)), n + n)
    return table, refs, holds, count


def exact(c, seed):
    if c["kind"] == "beam":
        return _exact_beam(c, seed)
    pool = _arrays(c, None)
    _fill(c, seed, pool)
    if c["kind"] in ("fork", "compact"):
        table, refs, holds, last = _exact_tables(c, seed)
        holds = torch.tensor(holds, device=DEV)
        if c["kind"] == "compact":
            return [_i32(table), _i32(refs), _i32([last]), pool["k"][:, holds].double(), pool["v"][:, holds].double()]
        at = holds[torch.tensor(last, device=DEV)]
        k, v = pool["k"][:, at].double(), pool["v"][:, at].double()
        if c["q8"]:
            k = k * pool["ks"][:, at].double()[..., None]
            v = v.transpose(-1, -2).flatten(-3, -2) * pool["vs"][:, at].double()[..., None]
        return [_i32(table), _i32(refs), k, v]
    B, L, H, G, hd, R = c["batch"], c["layers"], c["heads"], c["kv_heads"], c["head_dim"], c["page_rows"]
    q, k, v = _tokens(c, seed)
    cos, sin = (t.double() for t in _rope_table(c))
    table, _ = _tables(c)
    n = sizes(c)

    def turned(x, where, f32):
        """The rotated rows; as the engine stores them with f32 (each product and sum rounded)."""
        r = (lambda t: t.float().double()) if f32 else (lambda t: t)
        y, a, b = torch.empty_like(x, dtype=torch.float64), x[..., 0::2].double(), x[..., 1::2].double()
        y[..., 0::2] = r(r(a * cos[where]) - r(b * sin[where]))
        y[..., 1::2] = r(r(b * cos[where]) + r(a * sin[where]))
        return y

    def eighth(x):
        """What an 8-bit row stands for: the values and scales are defined by fp32 operations."""
        a = x.float().abs().amax(dim=-1, keepdim=True).clamp_min(2.0 ** -100).double()
        return torch.round(((x * (127.0 / a).float().double()).float()).double()) * (a / 127.0).float().double()

    def rows_of(name, l, pages):
        x = pool[name][l][pages].double()
        if c["q8"]:
            if name == "v":
                x = x.transpose(-1, -2).flatten(-3, -2)
            x = x * pool[name + "s"][l][pages].double()[..., None]
        return x.transpose(0, 1).flatten(1, 2)  # [kv_heads][rows][head_dim]

    out = torch.empty(L, B, H * hd, dtype=torch.float64, device=DEV)
    picked = torch.full((L, B, G, c.get("keep", 1)), -1, dtype=torch.int32, device=DEV)
    new = [torch.empty(B, L, G, hd, dtype=torch.float64, device=DEV) for _ in range(2)]
    for l in range(L):
        for i in range(B):
            p = n[i] - 1
            pages = torch.tensor(table[i][:p // R + 1], device=DEV)
            K, V = rows_of("k", l, pages), rows_of("v", l, pages)
            kr, vr = turned(k[l, i].unflatten(-1, (G, hd)), p, True), v[l, i].unflatten(-1, (G, hd)).double()
            if c["q8"]:
                kr, vr = eighth(kr), eighth(vr)
            K[:, p], V[:, p] = kr, vr
            K, V = K[:, :p + 1], V[:, :p + 1]
            new[0][i, l], new[1][i, l] = kr, vr
            qr = turned(q[l, i].unflatten(-1, (H, hd)), p, False)
            qf = turned(q[l, i].unflatten(-1, (H, hd)), p, True)  # (what the scores of pages are defined by)
            for g in range(G):
                see = torch.ones(p + 1, dtype=torch.bool, device=DEV)
                if c["kind"] == "sparse":
                    score = torch.zeros(p // R, dtype=torch.float64, device=DEV)
                    lo, hi = pool["bounds"][l][pages[:p // R], g].double().unbind(dim=1)
                    for a in range(g * H // G, (g + 1) * H // G):
                        score += torch.where(qf[a] > 0, qf[a] * hi, qf[a] * lo).sum(dim=-1)
                    order = sorted(range(p // R), key=lambda j, s=score.tolist(): (-s[j], j))[:c["keep"] - 1]
                    order = sorted(order) + [p // R]
                    picked[l, i, g, :len(order)] = _i32(order)
                    see[:] = False
                    for j in order:
                        see[j * R:(j + 1) * R] = True
                heads = slice(g * (H // G), (g + 1) * (H // G))
                s = (qr[heads] @ K[g].t().contiguous()) / math.sqrt(hd)
                w = torch.softmax(s.masked_fill_(~see, -math.inf), dim=-1)
                out[l, i, heads.start * hd:heads.stop * hd] = (w @ V[g].contiguous()).reshape(-1)
    return [out] + ([picked] if c["kind"] == "sparse" else []) + new
