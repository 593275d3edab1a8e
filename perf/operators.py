"""The operators on many tokens and on the 8-bit cache, as they are timed: each in its plain form (elementary torch
operations in 32 bits) and, where `own` is true, through the public binding, leap_amd.attention.

A case is a dict of plain values:
  kind       "prompt": HipAttention.prompt_async, packed sequences of new tokens, causal, over the cache
             "tree": HipAttention.tree_async, a tree of drafted tokens a sequence, then tree_keep_async of one path
             "q8step": one token of every sequence on an 8-bit cache (step_async, or step_batched_async for a batch)
             "q8kv": rows quantised into an 8-bit cache and read back (kv_write_async, kv_read_async)
  heads, kv_heads, head_dim, theta   the model's head shape and RoPE base
  layers     layers the handle holds; a pass runs each of them once
  batch, tokens, fewest, ctx, shortest, len_seed   sequences; new tokens of each (fewest..tokens, the first has
             tokens); rows of each with its new tokens (shortest..ctx, the first has ctx); the seed they are drawn with
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


def _case(kind, model, layers, batch, tokens, ctx, fewest=None, shortest=None, len_seed=0, name=None):
    c = {"kind": kind, "heads": model[0], "kv_heads": model[1], "head_dim": model[2], "theta": model[3],
         "layers": layers, "batch": batch, "tokens": tokens, "fewest": tokens if fewest is None else fewest,
         "ctx": ctx, "shortest": ctx if shortest is None else shortest, "len_seed": len_seed}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a short question to a small model: the least work a prompt has
        _case("prompt", TINY, 22, 1, 40, 40, name="prompt-tinyllama-40"),
        # a long document, the whole native context of a request at once
        _case("prompt", L3_8B, 1, 1, 8192, 8192, name="prompt-llama3-8b-8192"),
        # a server admits eight conversations of all lengths at once
        _case("prompt", L3_8B, 2, 8, 2011, 2011, fewest=17, shortest=17, len_seed=3, name="prompt8-llama3-8b-ragged2011"),
        # a long prompt taken in pieces: the last piece, over what is cached already
        _case("prompt", L3_70B, 2, 1, 500, 7300, name="prompt-llama3-70b-500-of-7300"),
        # speculative decoding of a small model: eight drafted tokens on a short conversation
        _case("tree", TINY, 22, 1, 8, 258, name="tree-tinyllama-8-ctx258"),
        # the same at the benchmark's context with a wider tree
        _case("tree", L3_8B, 16, 1, 31, 4096, name="tree-llama3-8b-31-ctx4096"),
        # a batch of conversations with trees of all sizes on a large model's stage
        _case("tree", L3_70B, 2, 8, 64, 8192, fewest=5, shortest=900, len_seed=11, name="tree8-llama3-70b-64-ragged8192"),
        # decoding from an 8-bit cache: a short conversation, where a launch is all there is
        _case("q8step", TINY, 22, 1, 1, 256, name="q8step-tinyllama-ctx256"),
        # the benchmark's headline on an 8-bit cache
        _case("q8step", L3_8B, 32, 1, 1, 4096, name="q8step-llama3-8b-ctx4096"),
        # a server's batch of conversations of all lengths on an 8-bit cache
        _case("q8step", L3_8B, 4, 32, 1, 8192, shortest=300, len_seed=7, name="q8step32-llama3-8b-ragged8192"),
        # a few rows moved into an 8-bit cache and read back
        _case("q8kv", TINY, 4, 1, 61, 256, name="q8kv-tinyllama-61"),
        # a stored prefix brought back into an 8-bit cache, every layer of a stage
        _case("q8kv", L3_8B, 8, 1, 8192, 8192, name="q8kv-llama3-8b-8192"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "tree", "tree", "q8step", "q8step", "q8kv"])
    model = rng.choice([TINY, L3_8B, L2_7B, L3_70B])
    seed = rng.randrange(1 << 16)
    if kind == "prompt":
        batch, tokens = _log_int(rng, 1, 16), _log_int(rng, 1, 8192)
        cached = rng.random() < 0.4
        c = _case(kind, model, 1, batch, tokens, tokens + (_log_int(rng, 1, 8192) if cached else 0), len_seed=seed)
        # (a batch's padded scores stay within those of the largest listed prompt)
        while c["batch"] * c["heads"] * c["tokens"] * c["ctx"] > 32 * 8192 ** 2:
            cut = c["tokens"] // 4
            if c["batch"] > 1 and rng.random() < 0.5:
                c["batch"] //= 2
            else:
                c["ctx"], c["tokens"] = c["ctx"] - cut - 1, c["tokens"] - cut - 1
        c["fewest"] = max(0, int(c["tokens"] * rng.uniform(0, 0.6))) if rng.random() < 0.7 else c["tokens"]
        c["shortest"] = c["ctx"] if c["ctx"] == c["tokens"] or rng.random() < 0.5 else max(1, c["ctx"] // 4)
    elif kind == "tree":
        tokens, ctx = rng.randint(2, 64), _log_int(rng, 128, 16384 if model is not L2_7B else 4096)
        c = _case(kind, model, 1, _log_int(rng, 1, 8), tokens, ctx, fewest=rng.randint(1, tokens),
                  shortest=max(1, int(ctx * rng.uniform(0.1, 1))), len_seed=seed)
    elif kind == "q8step":
        ctx = _log_int(rng, 16, 65536 if model is not L2_7B else 8192)
        batch = 1 if rng.random() < 0.4 else min(_log_int(rng, 2, 64), max(2, (1 << 18) // ctx))
        c = _case(kind, model, 1, batch, 1, ctx, shortest=ctx if rng.random() < 0.3 else max(1, ctx // 10), len_seed=seed)
    else:
        rows = _log_int(rng, 1, 8192)
        c = _case(kind, model, rng.randint(1, 8), 1, rows, rows + rng.randint(0, 500))
    # as many of the model's layers as keep a pass under a tenth of the largest listed case's work
    if kind != "q8kv":
        w = work(c)
        c["layers"] = max(1, min(model[4], 32, int(min(2e8 / w["bytes"], 5e10 / w["flops"]))))
    return c


def _seq_len(c):
    return 1 << max(6, (c["ctx"] - 1).bit_length())


def sizes(c):
    """(new tokens, rows with them) of each sequence."""
    r = random.Random(c["len_seed"])
    n = [c["tokens"]] + [r.randint(c["fewest"], c["tokens"]) for _ in range(c["batch"] - 1)]
    if c["kind"] == "prompt" and c["ctx"] == c["tokens"]:
        return n, list(n)
    return n, [c["ctx"]] + [max(a, r.randint(c["shortest"], c["ctx"])) for a in n[1:]]


def _parents(c, seed):
    """A tree of drafted tokens for each sequence, packed: each node's parent is an earlier node, or -1 for the
    last token of the conversation; most drafts hang on a recent one."""
    r, out = random.Random(seed * 7919 + 17), []
    for n in sizes(c)[0]:
        out.append([max(-1, j - r.choice((1, 1, 2, 3, 5))) for j in range(n)])
    return out


def _paths(c, seed):
    """One root-to-node path of each tree: what a verifier accepts, ended by -1."""
    r, out = random.Random(seed * 104729 + 5), []
    for p in _parents(c, seed):
        node, path = r.randrange(len(p)), []
        while node >= 0:
            path.append(node)
            node = p[node]
        out.append(path[::-1] + [-1] * (c["tokens"] - len(path)))
    return out


def work(c):
    H, G, hd = c["heads"], c["kv_heads"], c["head_dim"]
    row = 2 * G * (hd + 4) if c["kind"].startswith("q8") else 8 * G * hd  # a K and a V row of the cache
    b = f = 0
    for n, rows in zip(*sizes(c)):
        if c["kind"] == "q8kv":
            b += 2 * n * (8 * G * hd + row)
            f += 4 * n * G * hd
            continue
        if not n:
            continue
        b += (rows - n) * row + n * (8 * H * hd + 8 * G * hd + row)
        seen = n * (rows - n) + n * (n + 1) // 2
        if c["kind"] == "tree":
            seen = n * (rows - n) + 4 * n  # a node sees its few ancestors
            b += 16 * n * G * hd // 4      # the accepted quarter's rows move
        f += 4 * seen * H * hd
    return {"bytes": b * c["layers"], "flops": f * c["layers"]}


# ---- inputs ----------------------------------------------------------------

def _gen(seed, *what):
    s = seed & 0xFFFFFFFF
    for w in what:
        s = (s * 1000003 + w + 12345) & 0x7FFFFFFFFFFF
    return torch.Generator(device=DEV).manual_seed(s)


def _tokens(c, seed):
    """q, k and v of the new tokens, [layers][tokens][...].  Queries of twice the keys' spread give scores with the
    few heavy rows that trained attention has."""
    n, L, hd = sum(sizes(c)[0]), c["layers"], c["head_dim"]
    g = _gen(seed, 2)
    q = torch.randn(L, n, c["heads"] * hd, device=DEV, generator=g) * 2.0
    k = torch.randn(L, n, c["kv_heads"] * hd, device=DEV, generator=g)
    v = torch.randn(L, n, c["kv_heads"] * hd, device=DEV, generator=g)
    return q, k, v


def _fill_f32(c, seed, which, out):
    """Cache rows, [batch][layers][seq_len][kv_dim]: unit keys, as after RoPE, and values."""
    return out.normal_(generator=_gen(seed, 3, which))


def _fill_q8(c, seed, which, out, scale):
    """Rows of an 8-bit cache: values of a normal spread whose largest is near 127, and scales of such rows."""
    g = _gen(seed, 4, which)
    for t in out.flatten(0, 1):  # (a layer at a time: the fp32 draw is four times the cache)
        t.copy_(torch.randn(t.shape, device=DEV, generator=g).mul_(45.0).round_().clamp_(-127, 127))
    scale.uniform_(2.0 / 127, 3.0 / 127, generator=g)


def _table(c):
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


class _DeviceArray:
    """An array in device memory of a handle, for torch.as_tensor."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


def _caches(c, h):
    """Key and value caches of a handle, or (h None) of the plain form: [batch][layers][seq_len][kv_dim] each; of the
    8-bit cache each followed by its scales, which lie as [batch][layers][kv_heads][seq_len] and are seen as
    [batch][layers][seq_len][kv_heads]."""
    B, L, S, G = c["batch"], c["layers"], _seq_len(c), c["kv_heads"]
    values, scales = (B, L, S, G * c["head_dim"]), (B, L, G, S)
    if c["kind"].startswith("q8"):
        kinds = ((values, "|i1", torch.int8), (scales, "<f4", torch.float32)) * 2
        ptrs = h.kv_q8_device_ptr(0, 0) if h else None
    else:
        kinds = ((values, "<f4", torch.float32),) * 2
        ptrs = h.kv_device_ptr(0, 0) if h else None
    if h:
        t = [torch.as_tensor(_DeviceArray(h, p, shape, typestr), device=DEV) for p, (shape, typestr, _) in zip(ptrs, kinds)]
    else:
        t = [torch.empty(shape, dtype=dtype, device=DEV) for shape, _, dtype in kinds]
    return [x.transpose(2, 3) if x.shape == scales else x for x in t]


def prepare(c, seed):
    """The caches filled as a program holds them when the tokens come (in a handle, for the framework's operators),
    and the tokens' buffers."""
    B, L, hd, G = c["batch"], c["layers"], c["head_dim"], c["kv_heads"]
    q8 = c["kind"].startswith("q8")
    h = None
    if own:
        from leap_amd.attention import HipAttention
        h = HipAttention(c["heads"], G, hd, _seq_len(c), n_layers=L, rope_theta=c["theta"], max_batch=B,
                         **({"cache": "q8"} if q8 else {}))
    st = {"c": c, "h": h, "caches": _caches(c, h), "table": _table(c)}
    if q8:
        for which in (0, 1):
            _fill_q8(c, seed, which, *st["caches"][2 * which:2 * which + 2])
    else:
        for which in (0, 1):
            _fill_f32(c, seed, which, st["caches"][which])
    n, rows = sizes(c)
    N = sum(n)
    st["qkv"] = q, k, v = _tokens(c, seed)
    st["out"] = torch.empty_like(q)
    pos = [t - m for t, m in zip(rows, n)]
    begin = [sum(n[:i]) for i in range(B + 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    st["begin"], st["pos"] = i32(begin), i32(pos)
    st["seq"] = torch.tensor([i for i in range(B) for _ in range(n[i])], dtype=torch.long, device=DEV)
    st["N"], st["max_n"], st["max_pos"], st["rows"] = N, max(n), max(rows) - 1, sum(rows)
    if c["kind"] == "tree":
        st["parent"] = i32([x for p in _parents(c, seed) for x in p])
        st["path"] = i32(_paths(c, seed))
    if c["kind"] == "q8kv":
        st["back"] = [torch.empty_like(k), torch.empty_like(v)]
    # where the new rows are: a slice of the caches, or their indexes
    if B == 1:
        st["new"] = [t[0, :, pos[0]:pos[0] + n[0]] for t in st["caches"]]
    else:
        S = _seq_len(c)
        st["at"] = torch.tensor([(i * L + l) * S + pos[i] + j for l in range(L) for i in range(B) for j in range(n[i])],
                                dtype=torch.long, device=DEV)
        st["at_scale"] = ((st["at"] // S)[:, None] * G + torch.arange(G, device=DEV)) * S + (st["at"] % S)[:, None]
    torch.cuda.synchronize()
    return st


# ---- one pass ---------------------------------------------------------------

def _new_rows(st):
    """The rows of the new tokens as the cache holds them after the call."""
    new = st["new"] if "new" in st else [
        torch.index_select(t.view(-1, t.shape[-1]), 0, st["at"]) if t.is_contiguous()
        else torch.take(t.transpose(2, 3), st["at_scale"]) for t in st["caches"]]
    if len(new) == 2:
        return list(new)
    hd = st["c"]["head_dim"]  # 8 bits: the values they stand for
    return [x.unflatten(-1, (-1, hd)) * s[..., None] for x, s in ((new[0], new[1]), (new[2], new[3]))]


def _run_own(st):
    c, h = st["c"], st["h"]
    kind, B = c["kind"], c["batch"]
    q, k, v = st["qkv"]
    out = st["out"]
    stream = torch.cuda.current_stream().cuda_stream
    begin, pos = st["begin"].data_ptr(), st["pos"].data_ptr()
    for l in range(c["layers"]):
        if kind == "q8kv":
            at = c["ctx"] - c["tokens"], c["ctx"]
            h.kv_write_async(0, l, *at, k[l].data_ptr(), v[l].data_ptr(), stream)
            h.kv_read_async(0, l, *at, st["back"][0][l].data_ptr(), st["back"][1][l].data_ptr(), stream)
            continue
        qkvo = (q[l].data_ptr(), k[l].data_ptr(), v[l].data_ptr(), out[l].data_ptr(), stream)
        if kind == "prompt":
            h.prompt_async(l, B, begin, pos, st["N"], st["max_n"], st["max_pos"], *qkvo)
        elif kind == "tree":
            h.tree_async(l, B, begin, pos, st["parent"].data_ptr(), st["N"], st["max_n"], st["max_pos"], *qkvo)
        elif B == 1:
            h.step_async(l, c["ctx"] - 1, *qkvo)
        else:
            h.step_batched_async(l, B, pos, st["max_pos"], *qkvo, total_rows=st["rows"])
    if kind == "q8kv":
        return st["back"]
    if kind == "tree":
        h.tree_keep_async(B, pos, st["path"].data_ptr(), c["tokens"], stream)
    return [out] + _new_rows(st)


def _ancestors(parent, begin, seq, n):
    """[tokens][n]: whether a node descends from node m of its tree, or is it."""
    N = parent.numel()
    local = torch.arange(N, device=DEV) - begin.long()[seq]
    sees = torch.arange(n, device=DEV) == local[:, None]
    up = torch.where(parent >= 0, parent.long() + begin.long()[seq], torch.full_like(seq, -1))
    steps = max(1, (n - 1).bit_length())
    for _ in range(steps):  # each doubling reaches twice as far up
        has = up >= 0
        to = up.clamp_min(0)
        sees = sees | (sees[to] & has[:, None])
        up = torch.where(has, up[to], up)
    return sees


def _quantize(x, hd):
    """int8 values and one scale per head row."""
    g = x.unflatten(-1, (-1, hd))
    a = g.abs().amax(dim=-1).clamp_min(2.0 ** -100)
    t = torch.full_like(a, 127.0)
    return torch.round(g * (t / a)[..., None]).to(torch.int8).flatten(-2), a / t


def _rotate(x, cs, sn):
    """Interleaved pairs of each head; x [..., tokens, heads, head_dim], cs and sn [tokens][head_dim / 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    cs, sn = cs[:, None], sn[:, None]
    return torch.stack((a * cs - b * sn, b * cs + a * sn), dim=-1).flatten(-2)


def _run_plain(st):
    c = st["c"]
    kind, B, L, H, G, hd = c["kind"], c["batch"], c["layers"], c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = st["qkv"]
    caches, seq = st["caches"], st["seq"]
    N, n, K = st["N"], st["max_n"], st["max_pos"] + 1
    first = st["begin"].long()[seq]
    j = torch.arange(N, device=DEV) - first   # a token's place in its sequence
    row = st["pos"].long()[seq] + j           # and its cache row
    if kind == "q8kv":
        for i, x in enumerate((k, v)):
            x8, s = _quantize(x, hd)
            caches[2 * i][0, :, row], caches[2 * i + 1][0, :, row] = x8, s
        return [(caches[i][0, :, row].unflatten(-1, (-1, hd)) * caches[i + 1][0, :, row][..., None]).flatten(-2)
                for i in (0, 2)]
    at = row
    if kind == "tree":
        sees = _ancestors(st["parent"], st["begin"], seq, n)
        at = st["pos"].long()[seq] + sees.sum(dim=-1) - 1
    cs, sn = st["table"][0][at], st["table"][1][at]
    q = _rotate(q.unflatten(-1, (H, hd)), cs, sn)
    k = _rotate(k.unflatten(-1, (G, hd)), cs, sn).flatten(-2)
    # the new rows into the cache ([batch][layers][rows]; the indexed dimensions come first)
    if len(caches) == 2:
        for t, x in zip(caches, (k, v)):
            t[seq, :, row] = x.transpose(0, 1)
        keys, vals = (t[:, :, :K].unflatten(-1, (G, hd)) for t in caches)
    else:
        for i, x in enumerate((k, v)):
            x8, s = _quantize(x, hd)
            caches[2 * i][seq, :, row], caches[2 * i + 1][seq, :, row] = x8.transpose(0, 1), s.transpose(0, 1)
        keys, vals = (caches[i][:, :, :K].unflatten(-1, (G, hd)).float() * caches[i + 1][:, :, :K, :, None] for i in (0, 2))
    # scores of padded sequences, [batch][layers][KV heads][tokens * q heads of one][rows]
    pad = torch.zeros(B, L, n, H, hd, device=DEV)
    pad[seq, :, j] = q.transpose(0, 1)
    pad = pad.unflatten(3, (G, H // G)).permute(0, 1, 3, 2, 4, 5).reshape(B, L, G, n * (H // G), hd)
    s = torch.matmul(pad, keys.permute(0, 1, 3, 4, 2).contiguous()).mul_(1.0 / math.sqrt(hd))
    t = torch.arange(K, device=DEV)
    see = torch.zeros(B, n, K, dtype=torch.bool, device=DEV)
    if kind == "tree":
        first_row = st["pos"].long()[seq]
        node = t - first_row[:, None]
        among = (node >= 0) & (node < n)
        see[seq, j] = (node < 0) | (among & torch.gather(sees, 1, node.clamp(0, n - 1)))
    else:
        see[seq, j] = t <= row[:, None]
    see[..., 0] |= ~see.any(dim=-1)  # padding looks at one row, and is left out below
    s = s.unflatten(3, (n, H // G)).masked_fill_(~see[:, None, None, :, None], -math.inf)
    p = torch.exp_(s.sub_(s.amax(dim=-1, keepdim=True)))
    total = p.sum(dim=-1)
    o = torch.matmul(p.flatten(3, 4), vals.permute(0, 1, 3, 2, 4).contiguous()).unflatten(3, (n, H // G)) / total[..., None]
    out = o[seq, :, :, j].transpose(0, 1).reshape(L, N, H * hd)  # [tokens][layers][KV heads][q heads of one][head_dim]
    if kind == "tree":  # the accepted path's rows move together, in order
        kept = st["path"] >= 0
        b, i = kept.nonzero(as_tuple=True)
        first_row = st["pos"].long()[b]
        for x in caches:
            x[b, :, first_row + i] = x[b, :, first_row + st["path"].long()[b, i]]
    return [out] + _new_rows(st)


def run(st):
    return _run_own(st) if own else _run_plain(st)


# ---- the same in 64 bits ----------------------------------------------------

def exact(c, seed):
    kind, B, L, H, G, hd = c["kind"], c["batch"], c["layers"], c["heads"], c["kv_heads"], c["head_dim"]
    n, rows = sizes(c)
    q, k, v = _tokens(c, seed)
    cos, sin = (t.double() for t in _table(c))
    caches = _caches(c, None)
    q8 = kind.startswith("q8")
    for which in (0, 1):
        if q8:
            _fill_q8(c, seed, which, *caches[2 * which:2 * which + 2])
        else:
            _fill_f32(c, seed, which, caches[which])

    def turned(x, where, f32):
        """The rotated rows; as the engine stores them with f32 (each product and sum rounded)."""
        r = (lambda t: t.float().double()) if f32 else (lambda t: t)
        y, a, b = torch.empty_like(x, dtype=torch.float64), x[..., 0::2].double(), x[..., 1::2].double()
        cw, sw = cos[where][:, None], sin[where][:, None]
        y[..., 0::2], y[..., 1::2] = r(r(a * cw) - r(b * sw)), r(r(b * cw) + r(a * sw))
        return y

    def eighth(x):
        """What an 8-bit row stands for: the values and scales are defined by fp32 operations."""
        a = x.float().abs().amax(dim=-1, keepdim=True).clamp_min(2.0 ** -100).double()
        return torch.round(((x * (127.0 / a).float().double()).float()).double()) * (a / 127.0).float().double()

    if kind == "q8kv":
        return [eighth(x.unflatten(-1, (G, hd)).double()).flatten(-2) for x in (k, v)]
    parents = _parents(c, seed) if kind == "tree" else None
    paths = _paths(c, seed) if kind == "tree" else None
    out, new = torch.empty(L, sum(n), H * hd, dtype=torch.float64, device=DEV), [[], []]
    for l in range(L):
        done = 0
        for i in range(B):
            m, p0 = n[i], rows[i] - n[i]
            here = slice(done, done + m)
            done += m
            see = torch.ones(m, rows[i], dtype=torch.bool, device=DEV).tril(p0)
            where = torch.arange(p0, rows[i], device=DEV)
            if parents:
                up = torch.zeros(m, m, dtype=torch.bool)
                for a in range(m):
                    if parents[i][a] >= 0:
                        up[a] = up[parents[i][a]]
                    up[a, a] = True
                see[:, p0:] = up.to(DEV)
                where = p0 + up.sum(dim=1).to(DEV) - 1
            kr, vr = turned(k[l, here].unflatten(-1, (G, hd)), where, q8), v[l, here].unflatten(-1, (G, hd)).double()
            if q8:
                kr, vr = eighth(kr), eighth(vr)
                old = [caches[w][i, l, :p0].unflatten(-1, (G, hd)).double() * caches[w + 1][i, l, :p0, :, None].double() for w in (0, 2)]
            else:
                old = [caches[w][i, l, :p0].unflatten(-1, (G, hd)).double() for w in (0, 1)]
            K, V = torch.cat((old[0], kr)), torch.cat((old[1], vr))
            qr = turned(q[l, here].unflatten(-1, (H, hd)), where, False)
            for a in range(H):
                s = (qr[:, a] @ K[:, a // (H // G)].t().contiguous()) / math.sqrt(hd)
                w = torch.softmax(s.masked_fill_(~see, -math.inf), dim=-1)
                out[l, here, a * hd:(a + 1) * hd] = w @ V[:, a // (H // G)].contiguous()
            if paths:
                for x in (kr, vr):
                    kept = [a for a in paths[i] if a >= 0]
                    x[:len(kept)] = x[kept].clone()
            for x, to in ((kr, new[0]), (vr, new[1])):
                to.append(x if q8 else x.flatten(-2))
    shape = (lambda t: torch.cat(t).reshape(L, sum(n), *t[0].shape[1:])) if B == 1 else torch.cat
    return [out] + [shape(t) for t in new]
