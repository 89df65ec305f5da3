"""The operators of the paged 4-bit key/value cache, as cases that can be timed and compared.

Five kinds, each a call (or the two or three calls that go together) of a serving program:

* ``append``  keys and values of a prompt chunk rotated, quantised and written to the pages, and read back;
* ``decode``  one token of every sequence: its key and value appended, attention over the whole cache;
* ``prompt``  attention of a chunk of queries over the cache that already holds their own keys and values;
* ``fork``    rows that continue a common prefix: pages shared, the last one copied, room for one more token reserved;
* ``retire``  finished rows give their pages back and the pool is compacted.

A token's head row is held as D/g groups: m = the group's minimum, s = (maximum - minimum) / 15 (both fp16) and 4-bit codes
n = rint((x - m) / s); it stands for m + n s.  16 tokens of one head are one tile of T = 16 D + 128 D/g bytes:

    K codes [16][D/2] | K (s, m) fp16 pairs [16][D/g] | V codes [16][D/2] | V (s, m) [16][D/g]

a page is [kv heads][page/16][T], the pool uint8 [layers, pages, kv heads, page/16, T].  Within a code row the bytes stand in
the order the kernels read them (``_order``).  Sizes are the repository's own configurations' (32 heads of 128, 8 x 520 and
32 x 1030 tokens) and generic ones: shared heads, ragged lengths, small pages, long contexts.
"""
import math
import os
import random
import sys

import torch

own = False


def listed():
    return [
        # a short prompt on the OPT-shaped heads, no rotation: a chat turn
        dict(name="append 2x77", kind="append", rows=2, heads=32, kv=32, dim=128, group=64, page=64, rope=False, seq=77, context=0, ragged=False),
        # 8 prompts of different lengths continuing cached prefixes, shared heads, small groups and pages
        dict(name="append 8x2048 ragged", kind="append", rows=8, heads=32, kv=8, dim=128, group=32, page=16, rope=True, seq=2048, context=1000, ragged=True),
        # interactive decoding: one sequence, short context, latency is everything
        dict(name="decode 1x77", kind="decode", rows=1, heads=32, kv=32, dim=128, group=64, page=64, rope=False, context=77, ragged=False, idle=0),
        # the LLaMA-2-7B workload: 32 sequences past 1024-token prompts
        dict(name="decode 32x1030", kind="decode", rows=32, heads=32, kv=32, dim=128, group=64, page=64, rope=True, context=1030, ragged=False, idle=0),
        # a server's batch: sequences of any length, heads of 64 shared by four, two rows of the batch empty
        dict(name="decode 24 ragged", kind="decode", rows=24, heads=32, kv=8, dim=64, group=32, page=16, rope=True, context=6001, ragged=True, idle=2),
        # one long document, shared heads: the work of eight heads split over the whole GPU
        dict(name="decode 1x100001", kind="decode", rows=1, heads=32, kv=8, dim=128, group=128, page=128, rope=True, context=100001, ragged=False, idle=0),
        # questions of different lengths behind a cached text
        dict(name="prompt 8x77 ragged", kind="prompt", rows=8, heads=32, kv=32, dim=128, group=64, page=64, rope=True, seq=77, context=1000, ragged=True),
        # a chunk of a long prompt, shared heads
        dict(name="prompt 4096 after 4096", kind="prompt", rows=1, heads=32, kv=8, dim=128, group=64, page=64, rope=True, seq=4096, context=4096, ragged=False),
        # 7 samples continue one prompt, 8 layers
        dict(name="fork 7", kind="fork", layers=8, kv=32, dim=128, group=64, page=64, width=16, sources=1, forks=7, context=520, spare=16),
        # 64 rows continue 8 prompts, a 32-layer pool
        dict(name="fork 64", kind="fork", layers=32, kv=8, dim=128, group=32, page=64, width=40, sources=8, forks=64, context=1000, spare=64),
        # 3 of 8 rows are done
        dict(name="retire 3 of 8", kind="retire", layers=8, kv=32, dim=128, group=64, page=64, width=16, rows=8, gone=3, context=520, spare=8),
        # half of a batch of ragged rows is done, a 32-layer pool
        dict(name="retire 32 of 64", kind="retire", layers=32, kv=8, dim=128, group=128, page=32, width=80, rows=64, gone=32, context=600, spare=20),
    ]


def _log(rng, lo, hi):
    return int(min(max(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))), lo), hi))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "decode", "prompt", "prompt", "fork", "retire"))
    dim = rng.choice((64, 128, 128))
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    page = rng.choice((16, 32, 64, 128))
    if kind in ("append", "decode", "prompt"):
        heads = rng.choice((16, 20, 24, 32, 32, 40))
        kv = heads // rng.choice([r for r in (1, 2, 4, 5, 8) if heads % r == 0])
        c = dict(kind=kind, rows=_log(rng, 1, 48), heads=heads, kv=kv, dim=dim, group=group, page=page, rope=rng.random() < 0.6,
                 context=_log(rng, 1, 40000), ragged=rng.random() < 0.5)
        if kind == "decode":
            c["context"] = min(c["context"], max(1, 32 * 32 * 1030 // (c["rows"] * kv)))
            c["idle"] = rng.choice((0, 0, 1)) if c["rows"] > 1 else 0
        elif kind == "append":
            c["seq"] = min(_log(rng, 1, 4096), max(1, 8 * 2048 * 8 // (c["rows"] * kv)))
            c["context"] = min(c["context"], 5000)
        else:
            c["seq"] = _log(rng, 2, 4096)
            c["context"] = min(c["context"], max(1, 600000 // (c["rows"] * kv)))
            while c["rows"] * heads * c["seq"] * (c["seq"] + c["context"]) > 32 * 4096 * 8192:
                c["seq"] = max(1, c["seq"] // 2)
        return c
    c = dict(kind=kind, layers=rng.randint(1, 16), kv=rng.choice((4, 8, 16, 32)), dim=dim, group=group, page=page,
             context=_log(rng, 1, 1000))
    c["width"] = c["context"] // page + 2
    # (a pool of at most 600 MB)
    most = int(600e6 // (c["layers"] * c["kv"] * page * (dim + 8 * dim // group)))
    if kind == "fork":
        c["sources"] = rng.randint(1, max(1, min(8, most // (2 * c["width"]))))
        c["forks"] = _log(rng, 1, max(1, min(64, most - c["sources"] * c["width"] - 8) // 2))
        c["spare"] = rng.randint(1, 8)
    else:
        c["rows"] = rng.randint(2, max(2, min(64, most // c["width"])))
        c["gone"] = rng.randint(1, c["rows"] - 1)
        c["spare"] = rng.randint(0, 8)
    return c


# ---- sizes that follow from a case ----

def _tile_bytes(case):
    return 16 * case["dim"] + 128 * case["dim"] // case["group"]


def _contexts(case):
    """Tokens already cached, by row; -1: a row without a sequence.  Spread over the logarithm where they are ragged."""
    rows, most = case["rows"], case["context"]
    rng = random.Random(1000 * rows + most)
    n = [_log(rng, 1, max(most, 1)) if case["ragged"] and most else most for _ in range(rows)]
    if case["ragged"]:
        n[rng.randrange(rows)] = most
    for i in rng.sample(range(rows), case.get("idle", 0)):
        n[i] = -1
    return n


def _counts(case):
    """New tokens by row."""
    rows, seq = case["rows"], case["seq"]
    rng = random.Random(2000 * rows + seq)
    return [rng.randint(max(1, seq // 4), seq) if case["ragged"] and i else seq for i in range(rows)]


def _lengths(case):
    """Lengths of the rows of a pool (fork: of its sources)."""
    n = case["sources"] if case["kind"] == "fork" else case["rows"]
    rng = random.Random(3000 * n + case["context"])
    return [case["context"] if i == 0 else rng.randint(max(1, case["context"] // 2), case["context"]) for i in range(n)]


# ---- the format, in elementary torch operations ----

def _order(dim, group):
    """[16, T/16]: where in a tile the bytes of a token's row stand, for the row [K codes | K (s, m) | V codes | V (s, m)]
    with dim 2i in the low and 2i + 1 in the high half of code byte i."""
    half, par = dim // 2, 4 * dim // group
    row = torch.arange(16).unsqueeze(1)
    i = torch.arange(half).unsqueeze(0)
    w = i // 4
    k = row * half + 4 * ((w % 4) * (dim // 32) + w // 4) + i % 4
    h = i // 2
    v = 2 * ((h % 8) * (dim // 32) + h // 8) + i % 2 + 0 * row
    if dim == 128:
        v = v ^ (((row >> 1) & 1) << 5)
    v = v + row * half
    p = row * par + torch.arange(par).unsqueeze(0)
    return torch.cat((k, 16 * half + p, 16 * (half + par) + v, 16 * (2 * half + par) + p), 1)


def _group_params(x, group):
    """x fp32 [..., D] (fp16 values) -> codes, s, m."""
    y = x.unflatten(-1, (-1, group))
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    s = ((hi - lo) / torch.full((), 15.0, device=x.device)).half().float()
    n = torch.where(s > 0, torch.round((y - lo) / s.clamp_min(1e-30)).clamp(0, 15), torch.zeros_like(y))
    return n, s, lo


def _rotate(x, cos, sin):
    """x fp32 [..., D], cos and sin [..., D]: rotate half."""
    d = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., d:], x[..., :d]), -1) * sin


def _row_bytes(x, group):
    """fp32 [..., D] (fp16 values) -> code bytes and (s, m) bytes of its rows."""
    n, s, m = _group_params(x, group)
    n = n.flatten(-2).to(torch.uint8)
    codes = n[..., 0::2] | (n[..., 1::2] << 4)
    return codes, torch.cat((s, m), -1).half().flatten(-2).contiguous().view(torch.uint8)


def _values(rows, dim, group):
    """uint8 [..., T/16] rows -> K, V fp32 [..., D]."""
    half, par = dim // 2, 4 * dim // group
    out = []
    for a in (0, half + par):
        c = rows[..., a:a + half]
        n = torch.stack((c & 15, c >> 4), -1).flatten(-2).float().unflatten(-1, (-1, group))
        p = rows[..., a + half:a + half + par].contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))
        out.append((n * p[..., :1] + p[..., 1:]).flatten(-2))
    return out


def _gather(pool, table, tokens, dim, group):
    """The first `tokens` tokens of every row: K, V fp32 [B, kv, tokens, D]."""
    page = pool.shape[2] * 16
    order = _order(dim, group).to(pool.device).flatten()
    pages = pool[table[:, :(tokens + page - 1) // page].long().clamp_min(0)]         # [B, n, kv, page/16, T]
    rows = pages.transpose(1, 2).flatten(2, 3)[..., order].unflatten(-1, (16, -1)).flatten(2, 3)
    return _values(rows[:, :, :tokens], dim, group)


def _store(pool, table, at, k, v, valid, dim, group):
    """k, v fp32 [B, kv, S, D] to positions at [B, S] where valid; the others to the pool's last page, which no row holds."""
    page = pool.shape[2] * 16
    spare = pool.shape[0] - 1
    at = at.clamp_min(0)
    pid = torch.where(valid, table.gather(1, (at // page).clamp_max(table.shape[1] - 1)), spare).long()        # [B, S]
    order = _order(dim, group).to(pool.device)
    kb, kp = _row_bytes(k, group)
    vb, vp = _row_bytes(v, group)
    rows = torch.cat((kb, kp, vb, vp), -1).transpose(1, 2)                                 # [B, S, kv, T/16]
    kv, T = pool.shape[1], pool.shape[3]
    tile = (pid.unsqueeze(-1) * kv + torch.arange(kv, device=pool.device)) * (page // 16) + (at % page // 16).unsqueeze(-1)
    pool.view(-1)[tile.unsqueeze(-1) * T + order[at % 16].unsqueeze(2)] = rows


# ---- inputs ----

def _keys_values(gen, *shape):
    """Keys with some strong channels, as rotary models have them; values around zero."""
    k = torch.randn(shape, device="cuda", generator=gen)
    strong = torch.randn((shape[1], 1, shape[-1]), device="cuda", generator=gen)
    return (k + 2 * strong * (strong.abs() > 1.5)).half(), torch.randn(shape, device="cuda", generator=gen).half()


def _rope(positions, dim):
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, device="cuda").float() / dim))
    ang = torch.outer(torch.arange(positions, device="cuda").float(), inv)
    ang = torch.cat((ang, ang), -1)
    return ang.cos().half(), ang.sin().half()


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prepare_pool(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    fork = case["kind"] == "fork"
    lens, page, width = _lengths(case), case["page"], case["width"]
    rows = len(lens) + (case["forks"] if fork else 0)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + case["spare"] + (2 * case["forks"] if fork else 0) + (len(lens) if fork else 0)
    ids = rng.sample(range(pages), sum(need))
    table, refs = [], [0] * pages
    for i in range(rows):
        mine = [ids.pop() for _ in range(need[i])] if i < len(lens) else []
        for p in mine:
            refs[p] = 1
        table.append(mine + [-1] * (width - len(mine)))
    words = case["layers"] * pages * case["kv"] * page // 16 * _tile_bytes(case) // 8
    pool = torch.randint(-2 ** 62, 2 ** 62, (words,), device="cuda", generator=gen)
    state = dict(case=case, pool=pool.view(torch.uint8).view(case["layers"], pages, case["kv"], page // 16, _tile_bytes(case)),
                 lens=_int(lens + [0] * (rows - len(lens))))
    if fork:
        dst = list(range(len(lens), rows))
        rng.shuffle(dst)
        state.update(src=_int([rng.randrange(len(lens)) for _ in dst]), dst=_int(dst), ones=torch.ones(rows, dtype=torch.int32, device="cuda"))
    else:
        gone = rng.sample(range(rows), case["gone"])
        left = [r for r in range(rows) if r not in gone]
        if need[left[0]] > 1:                        # two of the rows that stay share their first page
            for r in left[1:2]:
                if lens[r] > page:
                    refs[table[r][0]] -= 1
                    table[r][0] = table[left[0]][0]
                    refs[table[r][0]] += 1
        used = {p for r in left for p in table[r] if p >= 0}
        state.update(gone=_int(gone), moves=sum(p >= len(used) for p in used))
    state.update(table=_int(table), refs=_int(refs))
    return state


def prepare(case, seed):
    if case["kind"] in ("fork", "retire"):
        return _prepare_pool(case, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    B, heads, kv, dim, group, page = (case[n] for n in ("rows", "heads", "kv", "dim", "group", "page"))
    pos = _contexts(case)
    counts = _counts(case) if "seq" in case else [1] * B
    seq = case.get("seq", 1)
    total = [p + c if p >= 0 else 0 for p, c in zip(pos, counts)]
    need = [(t + page - 1) // page for t in total]
    pages = sum(need) + 3
    ids = rng.sample(range(pages - 1), sum(need))           # the last page belongs to nobody
    table = [[ids.pop() for _ in range(n)] for n in need]
    width = max(need) + 1
    pool = torch.zeros(pages, kv, page // 16, _tile_bytes(case), dtype=torch.uint8, device="cuda")
    state = dict(case=case, pool=pool, table=_int([t + [-1] * (width - len(t)) for t in table]), pos=_int(pos), counts=None, rope=None)
    cached = total if case["kind"] == "prompt" else pos
    for i, n in enumerate(cached):
        for a in range(0, n, 16384):
            b = min(a + 16384, n)
            k, v = _keys_values(gen, 1, kv, b - a, dim)
            at = torch.arange(a, b, device="cuda").unsqueeze(0)
            _store(pool, state["table"][i:i + 1], at, k.float(), v.float(), at >= 0, dim, group)
    k, v = _keys_values(gen, B, kv, seq, dim)
    q = torch.randn(B, seq, heads * dim, device="cuda", generator=gen).half()
    state["qkv"] = torch.cat((q, k.transpose(1, 2).flatten(2), v.transpose(1, 2).flatten(2)), -1).contiguous()
    if case["ragged"] and "seq" in case:
        state["counts"] = _int(counts)
    if case["rope"]:
        state["rope"] = _rope(max(total) + 16, dim)
    if case["kind"] != "append":
        state["out"] = torch.randn(B, seq, heads * dim, device="cuda", generator=gen).half()
    if case["kind"] == "decode":
        state["qkv"], state["out"] = state["qkv"][:, 0], state["out"][:, 0]
    return state


# ---- one pass ----

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    return {"append": _append, "decode": _decode, "prompt": _prompt, "fork": _fork, "retire": _retire}[kind](state)


def _run_own(s):
    pkg = os.path.join(os.getcwd(), "sparse-quant_b200")      # the package `quant` lives in a folder whose name is not an identifier
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import quant
    case = s["case"]
    kind = case["kind"]
    if kind == "append":
        quant.kv4_append(s["qkv"], s["pool"], s["table"], s["pos"], case["heads"], rope=s["rope"], counts=s["counts"])
        k, v = quant.kv4_read(s["pool"], s["table"], s["pos"], case["seq"], counts=s["counts"])
        return dict(k=k, v=v)
    if kind == "decode":
        out = quant.kv4_decode_attention(s["qkv"], s["pool"], s["table"], s["pos"], case["heads"], rope=s["rope"], out=s["out"])
        k, v = quant.kv4_read(s["pool"], s["table"], s["pos"], 1)
        return dict(out=out, k=k, v=v)
    if kind == "prompt":
        return quant.kv4_attention(s["qkv"], s["pool"], s["table"], s["pos"], case["heads"], rope=s["rope"], counts=s["counts"], out=s["out"])
    table, lens, refs = s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    if kind == "fork":
        quant.kv4_fork(s["pool"], table, lens, refs, s["src"], s["dst"])
        pos = quant.kv4_reserve(table, lens, refs, s["ones"], case["page"])
        return dict(pool=s["pool"], table=table, lens=lens, refs=refs, pos=pos)
    quant.kv4_free(table, lens, refs, s["gone"])
    quant.kv4_compact(s["pool"], table, refs)
    return dict(pool=s["pool"], table=table, lens=lens, refs=refs)


def _heads(s, which):
    """The new tokens' queries, keys or values, fp32 [B, heads, S, D], and their positions [B, S] with what of them there is."""
    case = s["case"]
    x = s["qkv"] if s["qkv"].dim() == 3 else s["qkv"].unsqueeze(1)
    dim, n, kv = case["dim"], case["heads"], case["kv"]
    a = {"q": 0, "k": n * dim, "v": (n + kv) * dim}[which]
    x = x[..., a:a + (n if which == "q" else kv) * dim].unflatten(-1, (-1, dim)).transpose(1, 2).float()
    i = torch.arange(x.shape[2], device=x.device)
    at = s["pos"].unsqueeze(1) + i
    valid = (s["pos"] >= 0).unsqueeze(1) & (i < (x.shape[2] if s["counts"] is None else s["counts"].unsqueeze(1)))
    if s["rope"] is not None and which != "v":
        cos, sin = (t[at.clamp(0, t.shape[0] - 1)].float().unsqueeze(1) for t in s["rope"])
        x = _rotate(x, cos, sin)
    return x, at, valid


def _new_rows(s):
    case = s["case"]
    k, at, valid = _heads(s, "k")
    v, _, _ = _heads(s, "v")
    k = k.half().float()                                                        # keys reach the cache as fp16, as in the fp16 cache
    _store(s["pool"], s["table"], at, k, v, valid, case["dim"], case["group"])
    kv = []
    for x in (k, v):
        n, sc, m = _group_params(x, case["group"])
        kv.append(torch.where(valid[:, None, :, None], (n * sc + m).flatten(-2), torch.zeros_like(x)))
    return kv[0], kv[1], at, valid


def _append(s):
    k, v, _, _ = _new_rows(s)
    return dict(k=k.half(), v=v.half())


def _attend(s, q, at, valid):
    """softmax(q K^T / sqrt(D)) V over the cache, fp32; q [B, heads, S, D], at [B, S]."""
    case = s["case"]
    B, heads, S, dim = q.shape
    tokens = max(p + c for p, c in zip(_contexts(case), _counts(case) if "seq" in case else [1] * B))
    k, v = _gather(s["pool"], s["table"], tokens, dim, case["group"])
    q = q.reshape(B, case["kv"], -1, dim)                                      # the queries that share a head, one after the other
    p = (q @ k.transpose(-1, -2)) * dim ** -0.5
    hidden = torch.arange(tokens, device=q.device) > at.repeat(1, heads // case["kv"]).unsqueeze(-1)
    p = p.masked_fill_(hidden.unsqueeze(1), -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = ((p @ v) / total).reshape(B, heads, S, dim).transpose(1, 2).flatten(2)
    return torch.where(valid.unsqueeze(-1), out.half(), s["out"].view(B, S, -1))


def _decode(s):
    k, v, at, valid = _new_rows(s)
    q, _, _ = _heads(s, "q")
    return dict(out=_attend(s, q, at.clamp_min(0), valid)[:, 0], k=k.half(), v=v.half())


def _prompt(s):
    q, at, valid = _heads(s, "q")
    return _attend(s, q, at, valid)


def _free_first(refs):
    """Page numbers, the free ones first and in order."""
    return torch.argsort((refs != 0).to(torch.int8), stable=True).to(torch.int32)


def _fork(s):
    pool, page = s["pool"], s["case"]["page"]
    table, lens, refs = s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    src, dst = s["src"].long(), s["dst"].long()
    n = lens[src]
    full, part = n // page, (n % page > 0).int()
    rank = torch.where(part > 0, part.cumsum(0) - 1, part.sum() + (1 - part).cumsum(0) - 1)
    new = _free_first(refs)[rank]
    col = torch.arange(table.shape[1], device=table.device)
    old = table[src]
    rows = torch.where(col < full.unsqueeze(1), old, torch.where((col == full.unsqueeze(1)) & (part > 0).unsqueeze(1), new.unsqueeze(1), -1))
    table[dst], lens[dst] = rows, n
    refs.index_add_(0, rows.clamp_min(0).flatten().long(), (rows >= 0).flatten().int())
    last = old.gather(1, full.clamp_max(old.shape[1] - 1).unsqueeze(1).long())[:, 0].clamp_min(0).long()
    tile = torch.arange(page // 16, device=table.device) < ((n % page + 15) // 16).unsqueeze(1)
    pool[:, new.long()] = torch.where(tile[None, :, None, :, None], pool[:, last], pool[:, new.long()])
    # one more token for every row
    have = (lens + page - 1) // page
    more = (lens % page == 0).int()
    new = _free_first(refs)[(more.cumsum(0) - 1).clamp_min(0)]
    at = have.unsqueeze(1).long()
    table.scatter_(1, at, torch.where(more.unsqueeze(1) > 0, new.unsqueeze(1), table.gather(1, at)))
    refs.index_add_(0, new.long(), more)
    return dict(pool=pool, table=table, lens=lens + 1, refs=refs, pos=lens)


def _retire(s):
    pool = s["pool"]
    table, lens, refs = s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    gone = s["gone"].long()
    held = table[gone]
    refs.index_add_(0, held.clamp_min(0).flatten().long(), -(held >= 0).flatten().int())
    table[gone], lens[gone] = -1, 0
    used = refs > 0
    i = torch.arange(refs.shape[0], device=refs.device)
    low = i < used.sum()
    src, dst = (torch.argsort((~m).to(torch.int8), stable=True)[:s["moves"]] for m in (used & ~low, ~used & low))
    to = i.to(torch.int32).index_copy(0, src, dst.to(torch.int32))
    pool[:, dst] = pool[:, src]
    refs = refs.index_copy(0, dst, refs[src]).index_fill(0, src, 0)
    return dict(pool=pool, table=torch.where(table >= 0, to[table.clamp_min(0).long()], table), lens=lens, refs=refs)


# ---- the work of a pass ----

def work(case):
    row = case["kv"] * (_tile_bytes(case) // 16) if "kv" in case else 0          # bytes of a token's keys and values of one layer
    kind, dim = case["kind"], case["dim"]
    if kind in ("fork", "retire"):
        page = case["page"]
        if kind == "fork":
            lens = _lengths(case)
            mean = sum((n % page + 15) // 16 * 16 for n in lens) / len(lens)        # (which source a fork has depends on the seed)
            return dict(bytes=2 * mean * case["forks"] * row * case["layers"], flops=0)
        lens = _lengths(case)
        need = [(n + page - 1) // page for n in lens]
        kept = sum(need) * (case["rows"] - case["gone"]) / case["rows"]
        moved = kept * (1 - kept / (sum(need) + case["spare"]))                   # pages above the line that the kept ones fill
        return dict(bytes=2 * moved * page * row * case["layers"], flops=0)
    pos = _contexts(case)
    counts = _counts(case) if "seq" in case else [1] * case["rows"]
    live = [(p, c) for p, c in zip(pos, counts) if p >= 0]
    new = sum(c for _, c in live)
    if kind == "append":                                       # fp16 in, codes out; codes in and fp16 out to read back
        return dict(bytes=new * (4 * case["kv"] * dim + 2 * row) + case["rows"] * case["seq"] * 4 * case["kv"] * dim, flops=0)
    pairs = sum(c * p + c * (c + 1) // 2 for p, c in live)
    io = new * 2 * dim * (2 * case["heads"] + (2 * case["kv"] if kind == "decode" else 0))
    return dict(bytes=sum(p + c for p, c in live) * row + io, flops=4.0 * dim * case["heads"] * pairs)


# ---- the definition in 64 bits ----

def _nibble_places(dim):
    """For every dim: word of a K row and shift in it, half-word of a V row and shift in it."""
    d = torch.arange(dim, device="cuda")
    j = dim // 32
    return (d // 8 % 4) * j + d // 32, 4 * (d % 8), (d % 32 // 4) * j + d // 32, 4 * (d % 4)


def _exact_row(pool, table, tokens, dim, group):
    """K, V of one row of the table in 64 bits, [kv, tokens, D]."""
    page = pool.shape[2] * 16
    kw, ks, vw, vs = _nibble_places(dim)
    groups = torch.arange(dim, device="cuda") // group
    t = torch.arange(tokens, device="cuda")
    tiles = pool[table[t // page].long(), :, t % page // 16]                          # [tokens, kv, T]
    r = t % 16
    half, par = 8 * dim, 64 * dim // group
    pick = torch.arange(tokens, device="cuda")
    ck = tiles[..., :half].reshape(tokens, -1, 16, dim // 2)[pick, :, r].contiguous().view(torch.int32).long()
    pk = tiles[..., half:half + par].reshape(tokens, -1, 16, par // 16)[pick, :, r].contiguous().view(torch.float16).double()
    cv = tiles[..., half + par:2 * half + par].reshape(tokens, -1, 16, dim // 2)[pick, :, r].contiguous().view(torch.int16).long()
    pv = tiles[..., 2 * half + par:].reshape(tokens, -1, 16, par // 16)[pick, :, r].contiguous().view(torch.float16).double()
    if dim == 128:                                                                      # the 32-byte halves of these rows are exchanged
        swap = (r >> 1) & 1 == 1
        cv[swap] = torch.cat((cv[swap][..., 16:], cv[swap][..., :16]), -1)
    k = ((ck[..., kw] >> ks) & 15).double() * pk[..., 2 * groups] + pk[..., 2 * groups + 1]
    v = ((cv[..., vw] >> vs) & 15).double() * pv[..., 2 * groups] + pv[..., 2 * groups + 1]
    return k.transpose(0, 1), v.transpose(0, 1)


def _exact_turn(x, at, rope):
    if rope is None:
        return x
    a, b = x.chunk(2, -1)
    cos, sin = rope[0][at].double(), rope[1][at].double()
    (c0, c1), (s0, s1) = cos.chunk(2, -1), sin.chunk(2, -1)
    return torch.cat((a * c0 - b * s0, b * c1 + a * s1), -1)


def _exact_held(x, group):
    """What the cache holds for x [..., D] in 64 bits: steps and minima are fp16."""
    parts = []
    for y in x.split(group, -1):
        m = y.min(-1, keepdim=True).values
        s = ((y.max(-1, keepdim=True).values - m) / 15).to(torch.float16).double()
        n = torch.where(s > 0, torch.round((y - m) / torch.where(s > 0, s, torch.ones_like(s))).clamp(max=15), torch.zeros_like(y))
        parts.append(m + n * s)
    return torch.cat(parts, -1)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "retire"):
        return None                                              # whole numbers and moved bytes
    s = prepare(case, seed)
    B, heads, kv, dim, group = (case[n] for n in ("rows", "heads", "kv", "dim", "group"))
    x = s["qkv"] if s["qkv"].dim() == 3 else s["qkv"].unsqueeze(1)
    pos, S = s["pos"].tolist(), x.shape[1]
    counts = [S] * B if s["counts"] is None else s["counts"].tolist()
    new_k = torch.zeros(B, kv, S, dim, dtype=torch.float64, device="cuda")
    new_v = torch.zeros_like(new_k)
    out = None if kind == "append" else s["out"].double().view(B, S, heads, dim)
    for b in range(B):
        if pos[b] < 0:
            continue
        n, row = counts[b], x[b, :counts[b]].double().view(counts[b], -1, dim).transpose(0, 1)          # [heads + 2 kv, n, D]
        at = torch.arange(pos[b], pos[b] + n, device="cuda")
        if kind != "prompt":
            new_k[b, :, :n] = _exact_held(_exact_turn(row[heads:heads + kv], at, s["rope"]).half().double(), group)
            new_v[b, :, :n] = _exact_held(row[heads + kv:], group)
        if kind == "append":
            continue
        k, v = _exact_row(s["pool"], s["table"][b], pos[b] + n, dim, group)
        if kind == "decode":
            k[:, pos[b]], v[:, pos[b]] = new_k[b, :, 0], new_v[b, :, 0]
        q = _exact_turn(row[:heads], at, s["rope"])
        for h in range(heads):
            g = h // (heads // kv)
            sc = q[h] @ k[g].t() / math.sqrt(dim)
            sc.masked_fill_(torch.arange(pos[b] + n, device="cuda") > at.unsqueeze(1), -math.inf)
            out[b, :n, h] = torch.softmax(sc, -1) @ v[g]
    if kind == "append":
        return dict(k=new_k, v=new_v)
    out = out.flatten(2)
    return out if kind == "prompt" else dict(out=out[:, 0], k=new_k, v=new_v)
