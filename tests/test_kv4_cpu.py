"""The paged 4-bit key/value cache without a GPU: argument errors come back as status codes or RuntimeError before anything is
launched, and the oracle that the GPU tests use agrees with itself."""
import ctypes

import numpy as np
import pytest
import torch

import quant
from oracle import kv4


def test_tile_sizes():
    lib = quant.load_library()
    for D in (32, 64, 96, 128, 256):
        for G in (16, 32, 64, 128, 256):
            want = kv4.tile_bytes(D, G) if (D, G) in kv4.formats() else 0
            assert lib.w4a16_kv4_tile_bytes(D, G) == want
    assert len({kv4.tile_bytes(*f) for f in kv4.formats()}) == 5           # the format is told from a tile's size


def _p():
    buf = (ctypes.c_char * 4096)()
    return buf, (ctypes.addressof(buf) + 63) & ~63


def test_status_codes_of_cache_calls():
    lib = quant.load_library()
    keep, p = _p()

    def append(qkv=p, pool=p, table=p, pos=p, counts=None, cos=None, sin=None, batch=1, seq=1, heads=4, kv=2, D=128, g=64, page=16,
               pages=4, width=2, stride=8 * 128, rope_rows=0):
        return lib.w4a16_kv4_append(qkv, pool, table, pos, counts, cos, sin, batch, seq, heads, kv, D, g, page, pages, width, stride,
                                    rope_rows, None)

    def read(pool=p, table=p, pos=p, k=p, v=p, batch=1, seq=1, kv=2, D=128, g=64, page=16, pages=4, width=2):
        return lib.w4a16_kv4_read(pool, table, pos, None, k, v, batch, seq, kv, D, g, page, pages, width, None)

    def decode(qkv=p, pool=p, table=p, pos=p, cos=None, sin=None, out=p, ws=None, ws_bytes=0, batch=1, heads=4, kv=2, D=128, g=64, page=16, pages=4, width=2,
               stride=8 * 128, rope_rows=0):
        return lib.w4a16_kv4_decode_attention(qkv, pool, table, pos, cos, sin, out, ws, ws_bytes, batch, heads, kv, D, g, page, pages, width, stride,
                                              rope_rows, 0.1, None)

    def chunk(qkv=p, pool=p, table=p, pos=p, cos=None, sin=None, out=p, batch=1, seq=1, heads=4, kv=2, D=128, g=64, page=16, pages=4,
              width=2, stride=8 * 128, rope_rows=0):
        return lib.w4a16_kv4_attention(qkv, pool, table, pos, None, cos, sin, out, batch, seq, heads, kv, D, g, page, pages, width, stride,
                                       rope_rows, 0.1, None)

    for call in (append, decode, chunk):
        assert call(qkv=None) == 1 and call(pos=None) == 1 and call(cos=p) == 1 and call(sin=p) == 1
        assert call(heads=3) == 2 and call(stride=8 * 128 - 4) == 2 and call(cos=p, sin=p, rope_rows=0) == 2
        assert call(qkv=p + 2) == 4 and call(pos=p + 1) == 4
        assert call(heads=2 ** 24, kv=2 ** 20, stride=2 ** 40) == 9
    assert append(stride=7 * 128) == 2 and decode(stride=7 * 128) == 2 and chunk(stride=3 * 128) == 2
    for call in (append, read, decode, chunk):
        assert call(pool=None) == 1 and call(table=None) == 1
        assert call(g=16) == 3 and call(D=64, g=128) == 2 and call(D=96, g=32) == 2
        assert call(page=8) == 2 and call(page=48) == 2 and call(page=2048) == 2
        assert call(pages=0) == 2 and call(width=0) == 2 and call(kv=0) == 2 and call(batch=-1) == 2
        assert call(width=2 ** 26) == 9 and call(pool=p + 8) == 4
        assert call(batch=0) == 0                                              # nothing to do
    assert read(k=None) == 1 and read(v=p + 2) == 4
    assert decode(out=None) == 1 and chunk(out=p + 2) == 4
    # rows over a wide table are dealt to the whole GPU: that needs a workspace
    need = lib.w4a16_kv4_decode_workspace(1, 4, 2, 128, 64, 16, 10000)
    assert need > 0 and lib.w4a16_kv4_decode_workspace(64, 32, 32, 128, 64, 16, 2) == 0
    assert decode(width=10000) == 5 and decode(width=10000, ws=p, ws_bytes=need - 1) == 5 and decode(width=10000, ws=p + 2, ws_bytes=need) == 4
    assert append(seq=0) == 0 and read(seq=0) == 0 and chunk(seq=0) == 0
    assert append(seq=-1) == 2 and read(seq=-1) == 2 and chunk(seq=-1) == 2
    for call in (append, read, decode, chunk):
        assert call(batch=65536) == 9
    del keep


def test_status_codes_of_page_calls():
    lib = quant.load_library()
    keep, p = _p()

    def reserve(table=p, lens=p, refs=p, counts=p, pos=p, rows=2, width=2, pages=4, page=16):
        return lib.w4a16_kv4_reserve(table, lens, refs, counts, pos, rows, width, pages, page, None)

    def free(table=p, lens=p, refs=p, which=p, n=1, rows=2, width=2, pages=4):
        return lib.w4a16_kv4_free(table, lens, refs, which, n, rows, width, pages, None)

    def fork(pool=p, table=p, lens=p, refs=p, src=p, dst=p, ws=p, ws_bytes=4096, n=1, rows=2, width=2, layers=1, pages=4, kv=1, D=64, g=32,
             page=16):
        return lib.w4a16_kv4_fork(pool, table, lens, refs, src, dst, ws, ws_bytes, n, rows, width, layers, pages, kv, D, g, page, None)

    def compact(pool=p, table=p, refs=p, ws=p, ws_bytes=4096, rows=2, width=2, layers=1, pages=4, kv=1, D=64, g=32, page=16):
        return lib.w4a16_kv4_compact(pool, table, refs, ws, ws_bytes, rows, width, layers, pages, kv, D, g, page, None)

    for call in (reserve, free, fork, compact):
        assert call(table=None) == 1 and call(refs=None) == 1
        assert call(rows=0) == 2 and call(width=0) == 2 and call(pages=0) == 2
        assert call(table=p + 2) == 4 and call(refs=p + 2) == 4
        assert call(width=2 ** 27) == 9
    assert reserve(lens=None) == 1 and reserve(counts=None) == 1 and reserve(pos=None) == 1 and reserve(page=24) == 2
    assert reserve(rows=8193) == 9 and free(rows=2 ** 20, width=2 ** 11) == 9
    assert free(lens=None) == 1 and free(which=None) == 1 and free(n=-1) == 2 and free(n=0, which=None) == 0
    assert fork(pool=None) == 1 and fork(lens=None) == 1 and fork(src=None) == 1 and fork(dst=None) == 1 and fork(layers=0) == 2
    assert fork(n=-1) == 2 and fork(n=8193) == 9 and fork(g=48) == 3 and fork(pool=p + 4) == 4
    assert fork(ws=None) == 5 and fork(ws_bytes=lib.w4a16_kv4_fork_workspace(1, 2) - 1) == 5 and fork(n=0, src=None, dst=None) == 0
    assert compact(ws=None) == 5 and compact(ws_bytes=lib.w4a16_kv4_compact_workspace(4) - 1) == 5 and compact(layers=-1) == 2
    del keep


def test_python_entry_points_refuse_host_tensors_and_wrong_formats():
    with pytest.raises(RuntimeError, match="unsupported group size"):
        quant.kv4_pool(1, 4, 2, 128, group=48, device="cpu")
    for kw in (dict(head_dim=96), dict(head_dim=64, group=128), dict(head_dim=128, page_size=24), dict(head_dim=128, page_size=8)):
        with pytest.raises(RuntimeError):
            quant.kv4_pool(1, 4, 2, device="cpu", **kw)
    with pytest.raises(RuntimeError):
        quant.kv4_pool(1, 0, 2, 128, device="cpu")
    pool = quant.kv4_pool(2, 4, 2, 128, page_size=32, group=64, device="cpu")
    assert tuple(pool.shape) == (2, 4, 2, 2, 2304) and pool.dtype == torch.uint8 and not pool.any()
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 2, dtype=torch.int32)
    x = torch.zeros(1, 1, 8 * 128, dtype=torch.float16)
    for call in (lambda: quant.kv4_append(x, pool[0], t, i, 4), lambda: quant.kv4_read(pool[0], t, i, 1),
                 lambda: quant.kv4_decode_attention(x[0], pool[0], t, i, 4), lambda: quant.kv4_attention(x, pool[0], t, i, 4),
                 lambda: quant.kv4_reserve(t, i, i, i, 32), lambda: quant.kv4_free(t, i, i, i),
                 lambda: quant.kv4_fork(pool, t, i, i, i, i), lambda: quant.kv4_compact(pool, t, i)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()


@pytest.mark.parametrize("D,G", kv4.formats())
def test_oracle_format_round_trip(D, G):
    """Every byte of a tile belongs to one token's row, and a row reads back within half a step of what was stored."""
    seen = np.zeros(kv4.tile_bytes(D, G), dtype=int)
    pages = kv4.Pages(np.zeros((2, 1, 1, kv4.tile_bytes(D, G)), np.uint8), np.array([[1]]), D, G)
    rng = np.random.default_rng(D + G)
    for r in range(16):
        kb, vb, sh, kp, vp = pages._places(r)
        for at in (kb, vb):
            np.add.at(seen, at[sh == 0], 1)
        for p in kp + vp:
            seen[p:p + 4] += 1
        k, v = rng.standard_normal((2, D)).astype(np.float16)
        pages.store(0, 0, r, k, v)
        for x, y in zip((k, v), pages.load(0, 0, r)):
            assert np.array_equal(y, kv4.held(x, G))
            step = (x.reshape(-1, G).max(1) - x.reshape(-1, G).min(1)).astype(np.float64) / 15
            # half a step, and what rounding the step to fp16 (2^-11 of it) adds up to over 15 of them
            assert (np.abs(y - x).reshape(-1, G) <= step[:, None] * (0.5 + 15 * 2.0 ** -11)).all()
    assert (seen == 1).all()


def test_oracle_quantiser_edges():
    x = np.zeros((6, 64), np.float16)
    x[1] = 3.5                                       # constant: no step, read back exactly
    x[2, 5] = np.inf
    x[3, 7] = np.nan
    x[4, :32] = -65504
    x[4, 32:] = 65504                                # the widest range there is: the step still fits fp16
    x[5, 1] = 2.0 ** -24                             # the smallest: the step rounds to nothing
    y = kv4.held(x, 64)
    assert (y[0] == 0).all() and (y[1] == 3.5).all() and np.isnan(y[2]).all() and np.isnan(y[3]).all()
    assert np.abs(y[4] - x[4]).max() <= 65504 * 2 * 2.0 ** -11 and np.abs(y[5] - x[5].astype(float)).max() <= 2.0 ** -24


def test_oracle_pages():
    pool = np.arange(2 * 6 * 1 * 2 * 4, dtype=np.uint8).reshape(2, 6, 1, 2, 4)
    table, lens, refs = [[-1] * 3 for _ in range(3)], [0] * 3, [0] * 6
    assert kv4.reserve(table, lens, refs, [33, 0, 64], 32) == [0, -1, 0] and table[0][:2] == [0, 1] and table[2][:2] == [2, 3]
    assert kv4.reserve(table, lens, refs, [1, 96, 1], 32) == [33, -1, -1] and lens == [34, 0, 64]       # 3 + 1 pages wanted, 2 there
    kv4.fork(pool, table, lens, refs, [0, 0, 0], [1, 1, 2], 32)
    assert table[1] == [0, 4, -1] and refs == [2, 1, 1, 1, 1, 0] and (pool[:, 4, :, :1] == pool[:, 1, :, :1]).all() and lens[1] == 34
    kv4.free(table, lens, refs, [0, 0, 2])
    assert refs == [1, 0, 0, 0, 1, 0]
    want = pool[:, 4].copy()
    kv4.compact(pool, table, refs)
    assert table[1] == [0, 1, -1] and refs == [1, 1, 0, 0, 0, 0] and (pool[:, 1] == want).all()


def test_decoder_on_the_host_refuses_the_paged_cache():
    from w4a16.models import Decoder, DecoderConfig
    cfg = DecoderConfig("opt", layers=1, hidden=256, heads=4, ffn=512, vocab=64, group_size=128, max_positions=32, kv_bits=4)
    with pytest.raises(RuntimeError, match="GPU"):
        Decoder(cfg, device="cpu", seed=1).reset(1, 8)
    cfg.kv_bits = 8
    with pytest.raises(ValueError):
        Decoder(cfg, device="cpu", seed=1)
