"""The paged 4-bit key/value cache on the GPU against the oracle (oracle/kv4.py).

Append is compared byte for byte: quantisation and rotation are single fp32 operations in a fixed order.  Reading back rounds m + n s to
fp16 once: half a step, 2^-11 of the value (2^-25 below fp16's normal numbers), and the same again for the fp32 step in between.

Attention, against float64 on the same cache and the same rotated fp16 queries.  For one output, with p the weights:
  scores   D products and sums in fp32 (2^-24 each, in any order) of at most X = max_t sum |k||q|; the chunk kernel rounds k to fp16 too
           (2^-11 of X).  A score off by e moves every weight by e relative to the others: the output by at most 2 e max|v|.
  exp      2^-21 of a weight (ex2.approx with its scaled argument): 2 * 2^-21 max|v|
  weights  rounded to fp16 (2^-11), values to fp16 in the chunk kernel (2^-11): 2^-11 max|v| each.  The decode kernel weighs codes, of at
           most the group's range R = max - min instead of |v|: 2^-11 R, R <= 2 max|v|.
  output   rounded to fp16: 2^-11 of it.
Sums over n positions in fp32 add n 2^-24 max|v|."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _error_word():
    """Every test leaves the error word clear; those that raise it on purpose read and clear it themselves."""
    yield
    assert _take_error() == 0


def _take_error():
    import quant
    flag = ctypes.c_int(-1)
    assert quant.load_library().w4a16_device_error_flag(ctypes.byref(flag)) == 0
    if flag.value:
        assert quant.load_library().w4a16_device_error_clear() == 0
    return flag.value


def _rope(n, D, seed):
    ang = torch.rand(n, D // 2, generator=torch.Generator().manual_seed(seed)) * 6.28
    ang = torch.cat((ang, ang), -1)
    return ang.cos().half(), ang.sin().half()


class Case:
    """A cache of random rows with shuffled pages, in numpy (what the oracle holds) and on the device."""

    def __init__(self, lens, kv, heads, D, G, P, seed=0, new=1, rope=False, pad=0, scale_v=1.0, dead=()):
        rng = np.random.default_rng(seed)
        self.B, self.kv, self.heads, self.D, self.G, self.P, self.new = len(lens), kv, heads, D, G, P, new
        self.lens = [(-1 if b in dead else n) for b, n in enumerate(lens)]
        need = [0 if n < 0 else -(-(n + new) // P) for n in self.lens]
        pages = sum(need) + 2
        ids = list(rng.permutation(pages)[:sum(need)])
        width = max(need + [1]) + 1
        table = np.full((self.B, width), -1, np.int32)
        for b, n in enumerate(need):
            table[b, :n] = [ids.pop() for _ in range(n)]
        pool = rng.integers(0, 256, (pages, kv, P // 16, kv4.tile_bytes(D, G)), dtype=np.uint8)
        # unwritten tokens hold NaN scales: whatever reads past a length shows
        self.pages = kv4.Pages(pool, table, D, G)
        half, par = 8 * D, 64 * D // G
        for a in (half, 2 * half + par):
            pool[..., a:a + par] = np.frombuffer(np.float16([np.nan, np.nan]).tobytes() * (par // 4), np.uint8)
        for b, n in enumerate(self.lens):
            for t in range(max(n, 0)):
                for h in range(kv):
                    k, v = rng.standard_normal((2, D)).astype(np.float16)
                    self.pages.store(b, h, t, k, (v.astype(np.float32) * scale_v).astype(np.float16))
        x = rng.standard_normal((self.B, new, (heads + 2 * kv) * D + pad)).astype(np.float16)
        x[..., (heads + kv) * D:] *= np.float16(scale_v)
        self.qkv = torch.from_numpy(x)
        self.rope = _rope(width * P, D, seed) if rope else None

    def device(self):
        d = dict(qkv=self.qkv.cuda(), pool=torch.from_numpy(self.pages.pool).cuda(), table=torch.from_numpy(self.pages.table).cuda(),
                 pos=torch.tensor(self.lens, dtype=torch.int32).cuda())
        d["rope"] = None if self.rope is None else tuple(t.cuda() for t in self.rope)
        return d

    def part(self, b, i, which, head):
        """The (rotated) fp16 row of new token i."""
        at = {"q": 0, "k": self.heads, "v": self.heads + self.kv}[which]
        x = self.qkv[b, i].numpy()[(at + head) * self.D:(at + head + 1) * self.D]
        if self.rope is not None and which != "v":
            t = self.lens[b] + i
            x = kv4.rotate(x, self.rope[0][t].numpy(), self.rope[1][t].numpy())
        return x

    def append(self, counts=None):
        for b, n in enumerate(self.lens):
            for i in range(0 if n < 0 else self.new if counts is None else counts[b]):
                for h in range(self.kv):
                    self.pages.store(b, h, n + i, self.part(b, i, "k", h), self.part(b, i, "v", h))

    def attend(self, b, i, head, chunk, scale=None):
        """float64 output and its tolerance."""
        scale = self.D ** -0.5 if scale is None else scale
        K, V = self.pages.rows(b, head // (self.heads // self.kv), self.lens[b] + i + 1)
        q = self.part(b, i, "q", head).astype(np.float64)
        ref = kv4.attend(q, K, V, scale)
        if not len(K):
            return ref, np.zeros_like(ref)
        X = abs(scale) * (np.abs(K) @ np.abs(q)).max()
        big = np.abs(V).max()
        e = X * (self.D * 2.0 ** -23 + (2.0 ** -11 if chunk else 0))
        tol = big * (2 * e + 2 * 2.0 ** -21 + 2 * 2.0 ** -11 + len(K) * 2.0 ** -24) + 2.0 ** -11 * np.abs(ref) + 2.0 ** -24
        return ref, tol


def _bytes(t):
    return t.cpu().numpy()


@pytest.mark.parametrize("D,G", kv4.formats())
@pytest.mark.parametrize("rope", [False, True])
def test_append_writes_the_oracles_bytes(D, G, rope):
    import quant
    for P, lens, new, kv, pad, counts in ((16, [0, 5, 15, 16], 19, 2, 0, None), (64, [3, 0, 60], 9, 1, 8, [9, 0, 5]), (32, [0], 1, 3, 64, None)):
        c = Case(lens, kv, 2 * kv, D, G, P, seed=D + G + P, new=new, rope=rope, pad=pad, dead=(1,) if P == 64 else ())
        d = c.device()
        cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
        x = d["qkv"].clone()
        quant.kv4_append(d["qkv"], d["pool"], d["table"], d["pos"], c.heads, rope=d["rope"], counts=cnt)
        c.append(counts)
        assert np.array_equal(_bytes(d["pool"]), c.pages.pool)
        assert torch.equal(x, d["qkv"])
        k, v = quant.kv4_read(d["pool"], d["table"], d["pos"], new, counts=cnt)
        for b, n in enumerate(c.lens):
            m = 0 if n < 0 else new if counts is None else counts[b]
            for h in range(kv):
                for i in range(m):
                    for got, want in zip((k, v), c.pages.load(b, h, n + i)):
                        err = np.abs(got[b, h, i].double().cpu().numpy() - want)
                        assert (err <= 2.0 ** -11 * (1 + 2.0 ** -11) * np.abs(want) + 2.0 ** -25).all()
            assert not k[b, :, m:].any() and not v[b, :, m:].any()


def test_append_edges_of_the_quantiser():
    """Constant groups, the widest and the smallest ranges, infinities and NaN: the oracle's bytes (NaN scales compare as bytes too)."""
    import quant
    D, G = 128, 64
    c = Case([0], 1, 1, D, G, 16, new=7)
    x = c.qkv
    x[0, 0] = 2.5
    x[0, 1, :D:2], x[0, 1, 1:D:2] = -65504, 65504
    x[0, 2, 5] = float("inf")
    x[0, 2, D + 70] = float("-inf")
    x[0, 3, D + 3] = float("nan")
    x[0, 4, D:] = torch.linspace(0, 15 * 2.0 ** -24, 2 * D).half()
    x[0, 5, D:] *= 2.0 ** -14
    x[0, 6] = torch.arange(3 * D) % 16                         # codes exactly, ties nowhere
    x[0, 6, D:D + 64] = torch.arange(64) % 31 / 2.0 + 1        # step 1, half-way values: ties to even
    d = c.device()
    quant.kv4_append(d["qkv"], d["pool"], d["table"], d["pos"], 1)
    c.append()
    got, want = _bytes(d["pool"]), c.pages.pool
    nan = np.zeros_like(want, dtype=bool)
    half, par = 8 * D, 64 * D // G
    for a in (half, 2 * half + par):                           # a NaN scale may carry any payload; its minimum does not matter
        s = want[..., a:a + par].view(np.float16).reshape(*want.shape[:-1], -1, 2)
        g = got[..., a:a + par].copy().view(np.float16).reshape(*want.shape[:-1], -1, 2)
        assert np.array_equal(np.isnan(s[..., 0]), np.isnan(g[..., 0]))
        nan[..., a:a + par] = np.repeat(np.isnan(s[..., 0]), 4, -1)
    assert np.array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("D,G", kv4.formats())
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2), (5, 1), (16, 1), (24, 2)])
def test_decode_attention(D, G, heads, kv):
    import quant
    for rope, P, lens in ((False, 16, [0, 1, 15, 16, 17]), (True, 64, [63, 64, 200, 0]), (True, 32, [333])):
        c = Case(lens, kv, heads, D, G, P, seed=heads + P, rope=rope, pad=8 * (P == 64))
        d = c.device()
        out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], heads, rope=d["rope"])
        c.append()
        assert np.array_equal(_bytes(d["pool"]), c.pages.pool)
        got = out.double().cpu().numpy().reshape(c.B, heads, D)
        for b in range(c.B):
            for h in range(heads):
                ref, tol = c.attend(b, 0, h, chunk=False)
                assert (np.abs(got[b, h] - ref) <= tol).all(), (b, h, float(np.abs(got[b, h] - ref).max()), float(tol.max()))


@pytest.mark.parametrize("ctas", [-1, 1, 2, 3, 7, 64, 1000])
def test_decode_attention_dealt_to_ctas(ctas):
    """The work dealt to one CTA, to a few whose stretches begin and end inside rows, to more than there are chunks, or by units."""
    import quant
    lib = quant.load_library()
    try:
        lib.w4a16_tune_kv4(ctas)
        for D, G, heads, kv, lens in ((128, 64, 4, 2, [0, 15, 16, 129, 700]), (64, 32, 20, 2, [333, 0, 1]), (128, 128, 1, 1, [1100])):
            c = Case(lens, kv, heads, D, G, 32, seed=abs(ctas), rope=True, dead=(1,) if len(lens) == 3 else ())
            d = c.device()
            for again in range(2):
                out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], heads, rope=d["rope"])
                if not again:
                    c.append()
                assert np.array_equal(_bytes(d["pool"]), c.pages.pool)
                got = out.double().cpu().numpy().reshape(c.B, heads, D)
                for b in range(c.B):
                    for h in range(heads):
                        if c.lens[b] < 0:
                            assert not got[b, h].any()
                            continue
                        ref, tol = c.attend(b, 0, h, chunk=False)
                        assert (np.abs(got[b, h] - ref) <= tol).all(), (b, h, float(np.abs(got[b, h] - ref).max()), float(tol.max()))
    finally:
        lib.w4a16_tune_kv4(0)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
def test_decode_attention_scale(scale):
    import quant
    c = Case([70, 5], 2, 4, 64, 32, 16, seed=1)
    d = c.device()
    out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 4, scale=scale).double().cpu().numpy().reshape(2, 4, 64)
    c.append()
    for b in range(2):
        for h in range(4):
            ref, tol = c.attend(b, 0, h, chunk=False, scale=scale)
            assert (np.abs(out[b, h] - ref) <= tol).all()
    got = quant.kv4_attention(d["qkv"], d["pool"], d["table"], d["pos"], 4, scale=scale).double().cpu().numpy().reshape(2, 4, 64)
    for b in range(2):
        for h in range(4):
            ref, tol = c.attend(b, 0, h, chunk=True, scale=scale)
            assert (np.abs(got[b, h] - ref) <= tol).all()


def test_decode_attention_keeps_nan():
    """A query, a key or a value that is not finite makes the outputs NaN that depend on it, and no others."""
    import quant
    for what in ("q", "k", "v", "old"):
        c = Case([37, 50], 2, 4, 128, 64, 16, seed=2)
        x, D = c.qkv, 128
        if what == "old":
            for h in range(2):
                c.pages.store(0, h, 5, np.ones(D, np.float16), np.where(np.arange(D) == 70, np.inf, 1).astype(np.float16))
        else:
            at = {"q": 1, "k": 4, "v": 6}[what] * D                     # query head 1, key head 0, value head 0
            x[0, 0, at + 3] = float("nan") if what != "v" else float("inf")
        d = c.device()
        got = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 4).view(2, 4, D).isnan().cpu()
        want = torch.zeros_like(got)
        if what == "q":
            want[0, 1] = True
        elif what == "k":
            want[0, :2] = True
        elif what == "v":
            want[0, :2, :64] = True                                     # the group of dims that the infinity stands in
        else:
            want[0, :, 64:] = True
        assert torch.equal(got, want), what


def test_decode_attention_leaves_rows_without_a_sequence():
    import quant
    c = Case([40, 3, 7], 2, 4, 64, 32, 16, dead=(1,))
    d = c.device()
    out = torch.full((3, 4 * 64), 7.0, dtype=torch.float16, device="cuda")
    back = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 4, out=out)
    c.append()
    assert back is out and (out[1] == 7.0).all() and (out[0] != 7.0).any() and np.array_equal(_bytes(d["pool"]), c.pages.pool)
    fresh = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 4)
    assert not fresh[1].any() and torch.equal(fresh[::2], out[::2])


@pytest.mark.parametrize("scale_v", [1e-4, 1.0, 2000.0])
def test_decode_attention_values_of_any_size(scale_v):
    """Weights times value steps keep their precision for values near fp16's smallest and largest."""
    import quant
    c = Case([150, 90], 1, 2, 128, 64, 32, seed=3, scale_v=scale_v)
    # a run of rows a thousand times the others' size, and one of zeros
    for t in range(40, 60):
        c.pages.store(0, 0, t, np.ones(128, np.float16), (np.random.default_rng(t).standard_normal(128) * min(30 * scale_v, 15000)).astype(np.float16))
    for t in range(3):
        c.pages.store(0, 0, t, np.ones(128, np.float16), np.zeros(128, np.float16))
    d = c.device()
    out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 2).double().cpu().numpy().reshape(2, 2, 128)
    c.append()
    for b in range(2):
        for h in range(2):
            ref, tol = c.attend(b, 0, h, chunk=False)
            assert (np.abs(out[b, h] - ref) <= tol).all(), (float(np.abs(out[b, h] - ref).max()), float(tol.max()))


@pytest.mark.parametrize("size", [1e-5, 200.0])
def test_decode_attention_scores_of_any_size(size):
    """Large scores (one position takes all the weight, others underflow) and queries near fp16's smallest."""
    import quant
    c = Case([130], 2, 4, 128, 32, 16, seed=9)
    c.qkv[..., :4 * 128] *= size
    d = c.device()
    out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"], d["table"], d["pos"], 4).double().cpu().numpy().reshape(4, 128)
    c.append()
    for h in range(4):
        ref, tol = c.attend(0, 0, h, chunk=False)
        assert (np.abs(out[h] - ref) <= tol).all(), (float(np.abs(out[h] - ref).max()), float(tol.max()))


def test_decode_attention_long_sequence_and_one_head():
    """One head's 5000 positions are split over many CTAs and joined; checked with torch in float64 on what the cache reads back to."""
    import quant
    for heads, kv, D, G, P, n in ((1, 1, 128, 64, 64, 5001), (8, 1, 64, 32, 16, 4096), (12, 4, 128, 128, 128, 9000)):
        g = torch.Generator(device="cuda").manual_seed(n)
        need = n // P + 1
        pool = quant.kv4_pool(1, need + 1, kv, D, P, G)
        table = torch.randperm(need, device="cuda", generator=g).int().view(1, -1)
        x = torch.randn(1, n + 1, (heads + 2 * kv) * D, device="cuda", generator=g).half()
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        quant.kv4_append(x[:, :n].contiguous(), pool[0], table, zero, heads)
        pos = torch.full((1,), n, dtype=torch.int32, device="cuda")
        out = quant.kv4_decode_attention(x[:, n], pool[0], table, pos, heads).double().view(heads, D)
        k, v = quant.kv4_read(pool[0], table, zero, n + 1)
        q = x[0, n, :heads * D].view(heads, D).double()
        k, v = (t[0].double().repeat_interleave(heads // kv, 0) for t in (k, v))
        sc = (k @ q.unsqueeze(-1))[..., 0] * D ** -0.5
        ref = (torch.softmax(sc, -1).unsqueeze(1) @ v)[:, 0]
        # as at the head of this file, with keys and values read back to fp16 (2^-11 each)
        X = float((k.abs() @ q.abs().unsqueeze(-1)).max()) * D ** -0.5
        big = float(v.abs().max())
        tol = big * (2 * X * (2.0 ** -11 + D * 2.0 ** -23) + 4 * 2.0 ** -11 + n * 2.0 ** -24) + 2.0 ** -11 * ref.abs()
        assert ((out - ref).abs() <= tol).all()


@pytest.mark.parametrize("D,G", kv4.formats())
@pytest.mark.parametrize("heads,kv,new,lens,counts", [
    (2, 2, 1, [0, 30], None), (4, 2, 7, [0, 9, 100], [7, 0, 3]), (3, 1, 40, [17, 0], None), (6, 2, 130, [0], None), (2, 1, 33, [200, 1], [33, 32]),
])
def test_chunk_attention(D, G, heads, kv, new, lens, counts):
    import quant
    for rope, P in ((False, 16), (True, 64)):
        c = Case(lens, kv, heads, D, G, P, seed=new + P, new=new, rope=rope, dead=(1,) if counts and counts[1] == 0 else ())
        c.append(counts)
        d = c.device()
        cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
        out = torch.full((c.B, new, heads * D), 7.0, dtype=torch.float16, device="cuda")
        quant.kv4_attention(d["qkv"], d["pool"], d["table"], d["pos"], heads, rope=d["rope"], counts=cnt, out=out)
        got = out.double().cpu().numpy().reshape(c.B, new, heads, D)
        for b, n in enumerate(c.lens):
            m = 0 if n < 0 else new if counts is None else counts[b]
            assert (got[b, m:] == 7.0).all()
            for i in sorted({0, 1, 2, m // 2, m - 2, m - 1} & set(range(m))):
                for h in range(heads):
                    ref, tol = c.attend(b, i, h, chunk=True)
                    assert (np.abs(got[b, i, h] - ref) <= tol).all(), (b, i, h, float(np.abs(got[b, i, h] - ref).max()), float(tol.max()))


def test_chunk_attention_masked_values_that_are_not_finite():
    """A value that is not finite reaches the queries that see its token, in the dims of its group, and no others; so does a key."""
    import quant
    D, heads = 128, 4
    for what in ("v", "k"):
        c = Case([150], 2, heads, D, 64, 16, seed=6, new=40)
        at = 4 * D if what == "k" else 6 * D
        c.qkv[0, 7, at + 3] = float("nan") if what == "k" else float("inf")     # token 157, head 0, the first group of dims
        c.append()
        d = c.device()
        got = quant.kv4_attention(d["qkv"], d["pool"], d["table"], d["pos"], heads).view(40, heads, D).isnan().cpu()
        want = torch.zeros_like(got)
        want[7:, :2, :64 if what == "v" else D] = True
        assert torch.equal(got, want), what
        for i in (0, 6):
            for h in range(heads):
                ref, tol = c.attend(0, i, h, chunk=True)
                out = quant.kv4_attention(d["qkv"], d["pool"], d["table"], d["pos"], heads).double().cpu().numpy().reshape(40, heads, D)
                assert (np.abs(out[i, h] - ref) <= tol).all()


@pytest.mark.parametrize("heads,kv,S,ctx,counts", [(4, 1, 300, 700, None), (3, 3, 129, 0, None), (40, 8, 77, 500, [77, 5, 1, 64]), (32, 2, 1000, 30, [1000, 777])])
def test_chunk_attention_long(heads, kv, S, ctx, counts):
    """Several blocks of rows and steps of tokens, checked with torch in float64 on what the cache reads back to."""
    import quant
    D, G, P, B = 128, 64, 64, 1 if counts is None else len(counts)
    g = torch.Generator(device="cuda").manual_seed(S)
    need = (ctx + S) // P + 1
    pool = quant.kv4_pool(1, B * need, kv, D, P, G)
    table = torch.randperm(B * need, device="cuda", generator=g).int().view(B, -1)
    x = torch.randn(B, ctx + S, (heads + 2 * kv) * D, device="cuda", generator=g).half()
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    quant.kv4_append(x, pool[0], table, zero, heads, counts=None if cnt is None else cnt + ctx)
    pos = zero + ctx
    out = quant.kv4_attention(x[:, ctx:].contiguous(), pool[0], table, pos, heads, counts=cnt).double().view(B, S, heads, D)
    k, v = quant.kv4_read(pool[0], table, zero, ctx + S, counts=None if cnt is None else cnt + ctx)
    for b in range(B):
        n = S if counts is None else counts[b]
        q = x[b, ctx:ctx + n, :heads * D].view(n, heads, D).transpose(0, 1).double()
        kk, vv = (t[b, :, :ctx + n].double().repeat_interleave(heads // kv, 0) for t in (k, v))
        sc = (q @ kk.transpose(1, 2)) * D ** -0.5
        sc.masked_fill_(torch.arange(ctx + n, device="cuda") > torch.arange(ctx, ctx + n, device="cuda").unsqueeze(1), -float("inf"))
        ref = (torch.softmax(sc, -1) @ vv).transpose(0, 1)
        # as at the head of this file; keys and values as the kernel rounds them, read back
        X = float((q.abs() @ kk.abs().transpose(1, 2)).max()) * D ** -0.5
        tol = float(vv.abs().max()) * (2 * X * (D * 2.0 ** -23 + 2.0 ** -11) + 4 * 2.0 ** -11 + (ctx + n) * 2.0 ** -24) + 2.0 ** -11 * ref.abs()
        assert ((out[b, :n] - ref).abs() <= tol).all(), float((out[b, :n] - ref).abs().max())
        assert float((out[b, :n] - ref).norm() / ref.norm()) <= 2e-3            # and far closer on average: rounding errors of both signs
        assert not out[b, n:].any()


def _chunk_against_torch(heads, kv, D, G, P, S, ctx, counts=None, spoil=(), hidden=()):
    """kv4_attention of S queries behind ctx[b] tokens (negative: no sequence) against torch in float64 on what the cache reads back to.  spoil: (row,
    token, kv head, group, 'k' or 'v') of the cache that are made not finite; hidden: (row, page of the row) whose table entry is none of the pool."""
    import quant
    B = len(ctx)
    g = torch.Generator(device="cuda").manual_seed(S + sum(ctx))
    width = (max(ctx) + S) // P + 3
    pool = quant.kv4_pool(1, B * width, kv, D, P, G)
    table = torch.randperm(B * width, device="cuda", generator=g).int().view(B, -1)
    n = [0 if c < 0 else c + (S if counts is None else counts[b]) for b, c in enumerate(ctx)]
    x = torch.randn(B, max(n), (heads + 2 * kv) * D, device="cuda", generator=g).half()
    for b, t, h, gr, what in spoil:
        x[b, t, (heads + (kv if what == "v" else 0) + h) * D + gr * G + 1] = float("inf")
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    total = torch.tensor(n, dtype=torch.int32, device="cuda")
    quant.kv4_append(x, pool[0], table, zero, heads, counts=total)
    k, v = quant.kv4_read(pool[0], table, zero, max(n), counts=total)
    for b, p in hidden:
        table[b, p] = B * width + 5
    pos = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    q = torch.full((B, S, heads * D), float("nan"), dtype=torch.float16, device="cuda")      # (padding is not read)
    for b, c in enumerate(ctx):
        if c >= 0:
            q[b, :n[b] - c] = x[b, c:n[b], :heads * D]
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = quant.kv4_attention(q, pool[0], table, pos, heads, counts=cnt).view(B, S, heads, D)
    for b, c in enumerate(ctx):
        m = n[b] - max(c, 0)
        assert not out[b, m:].any()
        if m <= 0:
            continue
        qq = q[b, :m].view(m, heads, D).transpose(0, 1).double()
        kk, vv = (t[b, :, :n[b]].double().repeat_interleave(heads // kv, 0) for t in (k, v))
        sees = torch.arange(n[b], device="cuda") <= torch.arange(c, n[b], device="cuda").unsqueeze(1)
        for hb, p in hidden:
            if hb == b:
                sees[:, p * P:(p + 1) * P] = False
        bad_k = (~kk.isfinite()).any(-1).unsqueeze(1) & sees                    # [heads, 1 or m, tokens]
        bad_v = (sees.double() @ (~vv.isfinite()).double()) > 0                 # [heads, m, D]
        want_nan = (bad_v | bad_k.any(-1, keepdim=True)).transpose(0, 1)
        kk, vv = kk.nan_to_num(0, 0, 0), vv.nan_to_num(0, 0, 0)
        sc = (qq @ kk.transpose(1, 2)) * D ** -0.5
        sc.masked_fill_(~sees, -float("inf"))
        ref = (torch.softmax(sc, -1) @ vv).transpose(0, 1)
        got = out[b, :m].double()
        assert torch.equal(got.isnan(), want_nan)
        got, ref = got.masked_fill(want_nan, 0), ref.masked_fill(want_nan, 0)
        # as at the head of this file; keys and values as the kernel rounds them, read back
        X = float((qq.abs() @ kk.abs().transpose(1, 2)).max()) * D ** -0.5
        tol = float(vv.abs().max()) * (2 * X * (D * 2.0 ** -23 + 2.0 ** -11) + 4 * 2.0 ** -11 + n[b] * 2.0 ** -24) + 2.0 ** -11 * ref.abs()
        assert ((got - ref).abs() <= tol).all(), float((got - ref).abs().max())
        assert float((got - ref).norm()) <= 2e-3 * float(ref.norm())            # and far closer on average: rounding errors of both signs


@pytest.mark.parametrize("D,G", kv4.formats())
@pytest.mark.parametrize("heads,kv,S,ctx,counts", [
    (4, 4, 3, [1500], None), (8, 1, 20, [2100, 40, -1, 700], [20, 5, 0, 1]), (3, 1, 2, [511, 512, 513], None), (6, 2, 50, [0, 1100], None),
])
def test_chunk_attention_of_few_rows_over_many_tokens(D, G, heads, kv, S, ctx, counts):
    """The steps of a row tile are shared between CTAs, as many as its length asks for."""
    _chunk_against_torch(heads, kv, D, G, 64, S, ctx, counts)


@pytest.mark.parametrize("D,G", [(64, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("counts", [None, [3 - i % 4 for i in range(41)]])
def test_chunk_attention_of_ragged_batches(D, G, counts):
    """Rows much longer than the others, rows without a sequence, a wide table."""
    ctx = [3000 if i == 7 else 1700 if i == 30 else -1 if i % 11 == 5 else (37 * i) % 260 for i in range(41)]
    _chunk_against_torch(8, 4, D, G, 32, 3, ctx, counts)


@pytest.mark.parametrize("D,G", kv4.formats())
@pytest.mark.parametrize("ctx,counts", [([0, 300, 129], None), ([127, -1, 1000], [1100, 0, 250])])
def test_chunk_attention_of_many_rows(D, G, ctx, counts):
    """Two row tiles a CTA, whole and partly filled ones."""
    _chunk_against_torch(10, 2, D, G, 32, 1100, ctx, counts)


@pytest.mark.parametrize("heads,kv,S,ctx", [(4, 2, 5, [1300, 900]), (10, 2, 1100, [300, 0, 140])])
def test_chunk_attention_bad_values_and_pages_far_apart(heads, kv, S, ctx):
    """Values and keys that are not finite and pages that are none of the pool, in several steps of the same row; the rest stays as it is."""
    n = [c + S for c in ctx]
    spoil = [(0, 5, 0, 1, "v"), (0, 133, 1, 0, "v"), (0, n[0] - 2, 0, 0, "v"), (0, n[0] - 3, 1, 1, "k"), (1, 700, 1, 1, "v"), (1, 701, 1, 1, "v")]
    _chunk_against_torch(heads, kv, 128, 64, 32, S, ctx, spoil=spoil)
    assert _take_error() == 0
    _chunk_against_torch(heads, kv, 128, 64, 32, S, ctx, spoil=spoil[:1], hidden=[(0, 1), (0, 8), (1, 20)])
    assert _take_error() == 4


def test_chunk_attention_takes_queries_alone():
    """Rows of heads * head_dim elements: the queries without keys and values behind them."""
    import quant
    c = Case([20], 2, 4, 128, 64, 16, new=5)
    c.append()
    d = c.device()
    a = quant.kv4_attention(d["qkv"], d["pool"], d["table"], d["pos"], 4)
    b = quant.kv4_attention(d["qkv"][..., :4 * 128].contiguous(), d["pool"], d["table"], d["pos"], 4)
    assert torch.equal(a, b)


def test_positions_and_pages_out_of_range_raise_the_error_word():
    """Skipped by the kernels' own checks: nothing is written for them, the other rows are right."""
    import quant
    c = Case([20, 40], 1, 2, 64, 32, 16, seed=4)
    d = c.device()
    good = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"].clone(), d["table"], d["pos"], 2)
    width = d["table"].shape[1]
    for bad in (width * 16, 2 ** 31 - 1):
        pool, out = d["pool"].clone(), torch.full_like(good, 7.0)
        pos = torch.tensor([20, bad], dtype=torch.int32, device="cuda")
        quant.kv4_decode_attention(d["qkv"][:, 0], pool, d["table"], pos, 2, out=out)
        assert _take_error() == 3 and torch.equal(out[0], good[0]) and (out[1] == 7.0).all()
        quant.kv4_append(d["qkv"], pool, d["table"], pos, 2)
        assert _take_error() == 3
        k, _ = quant.kv4_read(pool, d["table"], pos, 1)
        assert _take_error() == 3 and not k[1].any()
        quant.kv4_attention(d["qkv"], pool, d["table"], pos, 2, out=out.view(2, 1, 128))
        assert _take_error() == 3 and (out[1] == 7.0).all()
    rope = tuple(t[:30].contiguous().cuda() for t in _rope(64, 64, 1))              # tables shorter than the second row's position
    out = torch.full_like(good, 7.0)
    quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"].clone(), d["table"], d["pos"], 2, rope=rope, out=out)
    assert _take_error() == 3 and (out[1] == 7.0).all() and (out[0] != 7.0).any()
    # a page of the second row that is none: its tokens are left out
    for page in (-1, d["pool"].shape[0], 2 ** 31 - 1):
        for col in (0, 2):
            table = d["table"].clone()
            table[1, col] = page
            e = Case([20, 40], 1, 2, 64, 32, 16, seed=4)
            e.pages.table = table.cpu().numpy()
            pool = d["pool"].clone()
            out = quant.kv4_decode_attention(d["qkv"][:, 0], pool, table, d["pos"], 2)
            assert _take_error() == 4 and torch.equal(out[0], good[0])
            e.pages.store(0, 0, 20, e.part(0, 0, "k", 0), e.part(0, 0, "v", 0))
            if col == 0:
                e.pages.store(1, 0, 40, e.part(1, 0, "k", 0), e.part(1, 0, "v", 0))
            assert np.array_equal(_bytes(pool), e.pages.pool)
            for h in range(2):
                ref, tol = e.attend(1, 0, h, chunk=True)
                assert (np.abs(out[1].double().cpu().numpy().reshape(2, 64)[h] - ref) <= tol).all()
            got = quant.kv4_attention(d["qkv"], pool, table, d["pos"], 2)
            assert _take_error() == 4
            for h in range(2):
                ref, tol = e.attend(1, 0, h, chunk=True)
                assert (np.abs(got[1, 0].double().cpu().numpy().reshape(2, 64)[h] - ref) <= tol).all()
    table = torch.full_like(d["table"], -1)                                          # nothing at all to attend to: zeros
    out = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"].clone(), table, d["pos"], 2)
    assert _take_error() == 4 and not out.any()


def test_argument_errors():
    import quant
    c = Case([20], 2, 4, 64, 32, 16)
    d = c.device()
    x, pool, table, pos = d["qkv"], d["pool"], d["table"], d["pos"]
    for call in (lambda: quant.kv4_append(x.float(), pool, table, pos, 4), lambda: quant.kv4_append(x, pool, table.long(), pos, 4),
                 lambda: quant.kv4_append(x, pool, table, pos.long(), 4), lambda: quant.kv4_append(x, pool, table, pos, 3),
                 lambda: quant.kv4_append(x, pool, table.expand(2, -1).contiguous(), pos, 4), lambda: quant.kv4_append(x[..., ::2], pool, table, pos, 2),
                 lambda: quant.kv4_append(x, pool.view(torch.int8), table, pos, 4), lambda: quant.kv4_append(x, pool[..., :-16].contiguous(), table, pos, 4),
                 lambda: quant.kv4_append(x, pool.unsqueeze(0), table, pos, 4), lambda: quant.kv4_append(x, pool, table, pos, 6),
                 lambda: quant.kv4_append(x, pool, table, pos, 4, rope=(torch.zeros(9, 32, dtype=torch.float16, device="cuda"),) * 2),
                 lambda: quant.kv4_append(x, pool, table, pos, 4, counts=torch.zeros(2, dtype=torch.int32, device="cuda")),
                 lambda: quant.kv4_decode_attention(x, pool, table, pos, 4), lambda: quant.kv4_decode_attention(x[:, 0], pool, table, pos, 4, out=x[:, 0]),
                 lambda: quant.kv4_attention(x, pool, table, pos, 4, out=x), lambda: quant.kv4_read(pool, table, pos, -1),
                 lambda: quant.kv4_fork(pool, table, pos, pos, pos, pos), lambda: quant.kv4_compact(pool[None], table, pos),
                 lambda: quant.kv4_reserve(table, pos, pos, pos, 17)):
        with pytest.raises(RuntimeError):
            call()


# ---- pages ----

def _book(rows, width, pages, layers=2, kv=2, D=64, G=32, P=32, seed=0):
    rng = np.random.default_rng(seed)
    pool = rng.integers(0, 256, (layers, pages, kv, P // 16, kv4.tile_bytes(D, G)), dtype=np.uint8)
    return dict(pool=pool, table=[[-1] * width for _ in range(rows)], lens=[0] * rows, refs=[0] * pages, P=P)


def _dev(book):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")          # noqa: E731
    return dict(pool=torch.from_numpy(book["pool"]).cuda(), table=i(book["table"]), lens=i(book["lens"]), refs=i(book["refs"]))


def _same(dev, book):
    assert dev["table"].tolist() == book["table"] and dev["lens"].tolist() == book["lens"] and dev["refs"].tolist() == book["refs"]
    assert np.array_equal(_bytes(dev["pool"]), book["pool"])


@pytest.mark.parametrize("rows,pages,width,P", [(3, 12, 6, 32), (40, 100, 20, 16), (1500, 3000, 9, 64)])
def test_pages_through_a_life(rows, pages, width, P):
    """Random reserves (also more than there is), forks (also refused ones), frees and compactions, step by step as the loops do."""
    import quant
    layers, kv = (2, 2) if rows < 100 else (1, 1)
    book = _book(rows, width, pages, layers, kv, P=P)
    dev = _dev(book)
    rng = np.random.default_rng(rows)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")          # noqa: E731
    ran_out = 0
    for step in range(30):
        counts = (rng.integers(-2, 2 * P, rows) * (rng.random(rows) < 0.5)).tolist()
        want = kv4.reserve(book["table"], book["lens"], book["refs"], counts, P)
        got = quant.kv4_reserve(dev["table"], dev["lens"], dev["refs"], i(counts), P)
        assert got.tolist() == want
        full = any(c > 0 and p < 0 for c, p in zip(counts, want))
        ran_out += full
        err = _take_error()
        assert (err in (3, 5)) == full
        _same(dev, book)
        n = int(rng.integers(1, rows + 2))
        src, dst = rng.integers(-1, rows + 1, n).tolist(), rng.integers(-1, rows + 1, n).tolist()
        kv4.fork(book["pool"], book["table"], book["lens"], book["refs"], src, dst, P)
        quant.kv4_fork(dev["pool"], dev["table"], dev["lens"], dev["refs"], i(src), i(dst))
        _take_error()
        _same(dev, book)
        gone = rng.integers(-1, rows + 1, int(rng.integers(1, max(2, rows // 2)))).tolist()
        kv4.free(book["table"], book["lens"], book["refs"], gone)
        quant.kv4_free(dev["table"], dev["lens"], dev["refs"], i(gone))
        assert _take_error() == (6 if any(not 0 <= r < rows for r in gone) else 0)
        _same(dev, book)
        if step % 3 == 2:
            kv4.compact(book["pool"], book["table"], book["refs"])
            quant.kv4_compact(dev["pool"], dev["table"], dev["refs"])
            _same(dev, book)
    assert ran_out


def test_forks_read_the_same_and_diverge():
    """Rows that continue a prefix see it through shared pages; what each appends afterwards is its own."""
    import quant
    D, G, P, kv, heads = 64, 32, 32, 2, 4
    pool = quant.kv4_pool(3, 20, kv, D, P, G)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")          # noqa: E731
    table, lens, refs = torch.full((4, 5), -1, dtype=torch.int32, device="cuda"), i([0] * 4), i([0] * 20)
    g = torch.Generator().manual_seed(0)
    n = 75
    pos = quant.kv4_reserve(table, lens, refs, i([n, 0, 0, 0]), P)
    assert pos.tolist() == [0, -1, -1, -1]
    x = torch.randn(4, n, (heads + 2 * kv) * D, generator=g).half().cuda()
    for layer in range(3):
        quant.kv4_append((x * (layer + 1)).contiguous(), pool[layer], table, pos, heads)
    quant.kv4_fork(pool, table, lens, refs, i([0, 0]), i([3, 1]))
    assert lens.tolist() == [n, n, 0, n] and table[:, :2].tolist() == [[0, 1]] * 2 + [[-1, -1]] + [[0, 1]] and table[:, 2].tolist() == [2, 4, -1, 3]
    zero = i([0, 0, -1, 0])
    for layer in range(3):
        k, v = quant.kv4_read(pool[layer], table, zero, n)
        assert torch.equal(k[1], k[0]) and torch.equal(v[3], v[0]) and k[0].abs().sum() > 0
    before = quant.kv4_read(pool[0], table, zero, n)
    pos = quant.kv4_reserve(table, lens, refs, i([1, 1, 0, 1]), P)
    assert pos.tolist() == [n, n, -1, n]
    y = torch.randn(4, (heads + 2 * kv) * D, generator=g).half().cuda()
    out = quant.kv4_decode_attention(y, pool[0], table, pos, heads)
    after = quant.kv4_read(pool[0], table, zero, n)
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
    k, _ = quant.kv4_read(pool[0], table, pos, 1)
    assert not torch.equal(k[0], k[1]) and not k[2].any()
    assert not torch.equal(out[0], out[1]) and not out[2].any()
    quant.kv4_free(table, lens, refs, i([0, 1]))
    quant.kv4_compact(pool, table, refs)
    k, v = quant.kv4_read(pool[0], table, i([-1, -1, -1, 0]), n)
    assert torch.equal(k[3], before[0][3]) and torch.equal(v[3], before[1][3]) and refs.tolist() == [1, 1, 1] + [0] * 17 and not k[0].any()
    quant.kv4_read(pool[0], table, i([0, -1, -1, 0]), n)                       # row 0 has no pages any more
    assert _take_error() == 4


# ---- streams, graphs, long offsets ----

def test_on_another_stream_and_captured():
    import quant
    c = Case([50, 70, 3], 2, 8, 128, 64, 16, rope=True)
    d = c.device()
    want = quant.kv4_decode_attention(d["qkv"][:, 0], d["pool"].clone(), d["table"], d["pos"], 8, rope=d["rope"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool = d["pool"].clone()
        got = quant.kv4_decode_attention(d["qkv"][:, 0], pool, d["table"], d["pos"], 8, rope=d["rope"])
    side.synchronize()
    assert torch.equal(want, got)
    # two captured steps, replayed on two streams at once: nothing of one call is shared with another
    graphs = []
    for k in range(2):
        s = dict(qkv=(d["qkv"] * (1 + k)).contiguous(), pool=d["pool"].clone())
        ref = quant.kv4_decode_attention(s["qkv"][:, 0], d["pool"].clone(), d["table"], d["pos"], 8, rope=d["rope"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = quant.kv4_decode_attention(s["qkv"][:, 0], s["pool"], d["table"], d["pos"], 8, rope=d["rope"])
        graphs.append((g, s, ref))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, (g, s, ref) in zip(streams, graphs):
            with torch.cuda.stream(st):
                s["out"].zero_()
                g.replay()
    torch.cuda.synchronize()
    for g, s, ref in graphs:
        assert torch.equal(s["out"], ref)


def test_calls_at_once_on_two_streams_and_from_two_graphs():
    """Token steps dealt over the whole GPU, chunks of few and of many rows: two programs at once, eager and captured, each with its own
    workspaces, give bit by bit what they give alone."""
    import quant
    programs = []
    for seed, heads, kv, D, G, n in ((1, 32, 8, 128, 64, 9000), (2, 16, 16, 64, 32, 7000)):
        g = torch.Generator(device="cuda").manual_seed(seed)
        width = n // 64 + 2
        pool = quant.kv4_pool(1, 2 * width, kv, D, 64, G)
        table = torch.randperm(2 * width, device="cuda", generator=g).int().view(2, -1)
        N = (heads + 2 * kv) * D
        x = torch.randn(2, n, N, device="cuda", generator=g).half()
        quant.kv4_append(x, pool[0], table, torch.zeros(2, dtype=torch.int32, device="cuda"), heads)
        pos = torch.tensor([n, n // 3], dtype=torch.int32, device="cuda")
        few, many = x[:, :9].contiguous(), x[:, :1500].contiguous()

        def run(pool=pool[0], table=table, pos=pos, heads=heads, one=x[:, 0].contiguous(), few=few, many=many):
            early = torch.clamp(pos - 2000, min=0)
            return (quant.kv4_decode_attention(one, pool, table, pos, heads), quant.kv4_attention(few, pool, table, pos - 10, heads),
                    quant.kv4_attention(many, pool, table, early, heads))
        programs.append(run)
    alone = [tuple(t.clone() for t in run()) for run in programs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in programs]
    for _ in range(3):
        got = []
        for st, run in zip(streams, programs):
            with torch.cuda.stream(st):
                got.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(alone, got) for a, b in zip(x, y))
    graphs, outs = [], []
    for st, run in zip(streams, programs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(run())
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(alone, outs) for a, b in zip(x, y))
    assert _take_error() == 0


def test_offsets_beyond_32_bits():
    """A layer of more than 4 GB: pages at its far end are written and read, those that 32-bit offsets would hit stay untouched."""
    import quant
    D, G, P, kv = 128, 32, 256, 32
    page_bytes = kv * P // 16 * kv4.tile_bytes(D, G)
    pages = (1 << 32) // page_bytes + 40
    pool = torch.empty((1, pages, kv, P // 16, kv4.tile_bytes(D, G)), dtype=torch.uint8, device="cuda")
    pool[:, :80].zero_()
    pool[:, -45:].zero_()
    far = pages - 3
    table = torch.tensor([[far, pages - 1]], dtype=torch.int32, device="cuda")
    i = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")          # noqa: E731
    x = torch.randn(1, 300, 3 * kv * D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    quant.kv4_append(x, pool[0], table, i(0), kv)
    assert not pool[0, :80].any() and pool[0, far].any() and pool[0, pages - 1].any()
    small = quant.kv4_pool(1, 2, kv, D, P, G)
    near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    quant.kv4_append(x, small[0], near, i(0), kv)
    assert torch.equal(small[0, 0], pool[0, far])
    for fn, arg in ((quant.kv4_decode_attention, x[:, 299]), (quant.kv4_attention, x[:, 299:].contiguous())):
        assert torch.equal(fn(arg, pool[0], table, i(299), kv), fn(arg, small[0], near, i(299), kv))
    a, b = quant.kv4_read(pool[0], table, i(0), 300), quant.kv4_read(small[0], near, i(0), 300)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # fork and compact over the same distance
    lens, refs = torch.tensor([300, 0], dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[0].long()] = 1
    refs[1:pages - 3] = 1                                             # only pages 0, far + 1 are free
    both = torch.cat((table, torch.full_like(table, -1)))
    quant.kv4_fork(pool, both, lens, refs, i(0), i(1))
    assert both[1].tolist() == [far, 0] and torch.equal(pool[0, 0, :, :3], pool[0, pages - 1, :, :3])
    refs[1:pages - 3] = 0
    quant.kv4_compact(pool, both, refs)
    assert both.tolist() == [[1, 2], [1, 0]] and refs[:4].tolist() == [1, 2, 1, 0] and torch.equal(pool[0, 1], small[0, 0])
