"""Decoder stacks on the paged 4-bit cache: the calls in the order a model makes them, against the same model with the cache calls
replaced by torch in float64 on what the cache reads back to."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _config(kind, heads=8):
    from w4a16.models import DecoderConfig
    if kind == "opt":
        return DecoderConfig("opt", layers=3, hidden=512, heads=heads, ffn=2048, vocab=1024, group_size=128, max_positions=512, kv_bits=4,
                             kv_group=32, kv_page=16)
    return DecoderConfig("llama", layers=3, hidden=512, heads=heads, ffn=1344, vocab=1024, group_size=64, max_positions=512, kv_bits=4)


def _rotated(x, pos, rope):
    if rope is None:
        return x
    cos, sin = (t[pos].double() for t in rope)
    h = x.shape[-1] // 2
    return (x * cos + torch.cat((-x[..., h:], x[..., :h]), -1) * sin).half().double()


def _plain_attention(qkv, pool, table, pos, heads, rope=None, scale=None, counts=None, out=None):
    import quant
    B, S = qkv.shape[:2]
    kv, D = pool.shape[1], quant.kv4._FORMATS[pool.shape[-1]][0]
    res = torch.zeros(B, S, heads * D, dtype=torch.float16, device="cuda")
    for b in range(B):
        p = int(pos[b])
        k, v = (t[0].double() for t in quant.kv4_read(pool, table[b:b + 1].contiguous(), torch.zeros_like(pos[b:b + 1]), p + S))
        for i in range(S):
            q = _rotated(qkv[b, i, :heads * D].view(heads, D).double(), p + i, rope)
            w = torch.softmax((k[:, :p + i + 1] @ q.unsqueeze(-1))[..., 0] * D ** -0.5, -1)
            res[b, i] = (w.unsqueeze(1) @ v[:, :p + i + 1])[:, 0].reshape(-1).half()
    return res


def _plain_decode(qkv, pool, table, pos, heads, rope=None, scale=None, out=None):
    import quant
    quant.kv4_append(qkv.unsqueeze(1).contiguous(), pool, table, pos, heads, rope=rope)
    return _plain_attention(qkv.unsqueeze(1), pool, table, pos, heads, rope)[:, 0]


@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_stack_matches_plain_attention_over_the_same_cache(kind, monkeypatch):
    import quant
    from w4a16.models import Decoder
    model = Decoder(_config(kind), device="cuda", seed=5).mark_static()
    ids = torch.randint(0, 1024, (3, 41), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))

    def steps():
        model.reset(3, 80)
        outs = [model(ids[:, :30]), model(ids[:, 30:])]                # a prompt in two chunks
        tok = torch.tensor([[5], [6], [7]], device="cuda")
        pos_t = torch.full((1,), 41, dtype=torch.long, device="cuda")
        for _ in range(2):
            outs.append(model.step_static(tok, pos_t, None).float())
        model.pos = 43
        outs.append(model(tok))
        return outs

    a = steps()
    monkeypatch.setattr(quant, "kv4_attention", _plain_attention)
    monkeypatch.setattr(quant, "kv4_decode_attention", _plain_decode)
    b = steps()
    for x, y in zip(a, b):
        if x.shape[-1] == 1:
            assert (x == y).float().mean() >= 2 / 3                      # greedy tokens: near ties may fall the other way
        else:
            # the linears' fp16 roundings around an attention that agrees to fp16: as between the fp16 stacks and their dense form
            assert ((x.float() - y.float()).norm() / y.float().norm()).item() <= 2e-2


@pytest.mark.parametrize("kind,heads", [("opt", 8), ("llama", 4)])
def test_generate_captured_and_eager_give_the_same_tokens(kind, heads):
    from w4a16.models import Decoder
    model = Decoder(_config(kind, heads), device="cuda", seed=3).mark_static()
    ids = torch.randint(0, 1024, (5, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    graphed, _, _ = model.generate_graphed(ids, 9, use_graph=True)
    eager, _, _ = model.generate_graphed(ids, 9, use_graph=False)
    assert torch.equal(graphed, eager)
    one_by_one, _, _ = model.generate(ids, 9)
    assert (one_by_one == eager).float().mean().item() >= 0.75


@pytest.mark.parametrize("S0", [64, 75])
def test_rows_that_share_a_prefix(S0):
    """generate_shared against whole prompts row by row: the same caches by construction up to the linears' tile shapes."""
    from w4a16.models import Decoder
    model = Decoder(_config("llama"), device="cuda", seed=8).mark_static()
    g = torch.Generator(device="cuda").manual_seed(4)
    prefix, suffix = torch.randint(0, 1024, (1, S0), device="cuda", generator=g), torch.randint(0, 1024, (4, 13), device="cuda", generator=g)
    got = model.generate_shared(prefix, suffix, 5)
    kv = model.kv4
    full = S0 // 64
    assert got.shape == (4, 5) and kv.lens.tolist() == [0, 0, 0, 0, S0] and int((kv.refs > 0).sum()) == -(-S0 // 64) and int(kv.refs.max()) == 1
    assert (kv.table[:4] == -1).all() and (kv.table[4, :full] >= 0).all()
    before = kv.pool[:, kv.table[4, 0].long()].clone()
    kv.compact()
    assert kv.table[4, 0] == 0 and torch.equal(kv.pool[:, 0], before)
    whole, _, _ = model.generate_graphed(torch.cat((prefix.expand(4, -1), suffix), 1), 5, use_graph=False)
    assert (whole == got).float().mean().item() >= 0.75


def test_refusals():
    from w4a16.models import Decoder
    cfg = _config("opt")
    model = Decoder(cfg, device="cuda", seed=1)
    ids = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for call in (lambda: model.generate_shared(ids, ids, 1), lambda: model.generate_shared(ids[:1], ids[:, :0], 1),
                 lambda: model.generate_shared(ids[:1], ids, 0)):
        with pytest.raises(RuntimeError):
            call()
    cfg16 = _config("opt")
    cfg16.kv_bits = 16
    with pytest.raises(RuntimeError, match="kv_bits"):
        Decoder(cfg16, device="cuda", seed=1).generate_shared(ids[:1], ids, 1)
