"""Token generation with TinyLM over the 4-bit cache, against the model run whole in torch.

The cached model differs from the whole one by its 4-bit keys and values, so the whole run below quantises them
(in float64) as the cache does; what is left are the GEMMs' TF32X3 (2^-21 of each product) and the cache's codes
that fall on a tie between the two: logits agree to 2e-3 of their spread.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def quantised(x, group):
    g = x.double().unflatten(-1, (-1, group))
    zero = g.amin(-1, keepdim=True).half().double()
    scale = ((g.amax(-1, keepdim=True) - zero) / 15).half().double()
    code = torch.where(scale > 0, torch.round((g - zero) / scale.clamp(min=1e-30)), 0.0).clamp(0, 15)
    return (code * scale + zero).flatten(-2)


def whole(model, ids, group):
    """Logits after every token of one sequence, in float64 with 4-bit keys and values."""
    c = model.c
    p = {k: v.double() for k, v in model.p.items()}
    ln = lambda x, n: torch.nn.functional.layer_norm(x, (c.d,), p[n + "_g"], p[n + "_b"], c.ln_eps)  # noqa: E731
    n, d = len(ids), c.d // c.heads
    x = p["tok"][torch.tensor(ids, device="cuda")] + p["pos"][:n]
    for i in range(c.layers):
        w = "l%d." % i
        q, k, v = (ln(x, w + "ln1") @ p[w + "wqkv"] + p[w + "bqkv"]).view(n, 3, c.heads, d).unbind(1)
        k, v = quantised(k, group), quantised(v, group)
        s = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        if c.softmax1:
            s = torch.cat([s, torch.zeros(c.heads, n, 1, dtype=s.dtype, device="cuda")], -1)
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1)[..., :n], v).reshape(n, c.d)
        x = x + o @ p[w + "wo"] + p[w + "bo"]
        x = x + torch.relu(ln(x, w + "ln2") @ p[w + "w1"] + p[w + "b1"]) @ p[w + "w2"] + p[w + "b2"]
    return ln(x, "lnf") @ p["tok"].T


@pytest.mark.parametrize("softmax1,group", [(False, 64), (True, 32)])
def test_steps_agree_with_the_whole_model(dev, softmax1, group):
    from scratchtape_b200.generate import Generator
    from scratchtape_b200.lm import LmConfig, TinyLM
    from scratchtape_b200.matmul import TF32X3
    cfg = LmConfig(layers=2, d=128, heads=2, dff=256, t=40, batch=2, softmax1=softmax1, gemm_prec=TF32X3)
    model = TinyLM(cfg, "cuda", seed=3)
    model.params.mul_(1.5)
    gen = Generator(model, 3, group=group)
    prompts = [[5, 7, 200, 7, 7, 31, 9, 250, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10], [40], [0, 255, 17]]
    seqs = [list(p) for p in prompts]
    tokens = prompts
    for _ in range(12):
        got = gen.forward(tokens)
        for b in range(3):
            want = whole(model, seqs[b], group)[-1]
            assert (got[b].double() - want).abs().max() <= 2e-3 * (want.max() - want.min())
        tokens = [[int(v)] for v in got.argmax(1).tolist()]
        for s, t in zip(seqs, tokens):
            s += t
    dev.sync()


def test_generate_with_penalties_and_masks(dev):
    from scratchtape_b200.generate import Generator
    from scratchtape_b200.lm import LmConfig, TinyLM
    cfg = LmConfig(layers=1, d=128, heads=2, dff=256, t=32, batch=2)
    model = TinyLM(cfg, "cuda", seed=1)
    prompts = [[1, 2, 3], [9, 8, 7, 6]]
    words = torch.zeros((2, 8), dtype=torch.int32)
    words[0] = -1                      # the first sequence: anything
    words[1, 2] = 0b1111 << 5          # the second: tokens 69 .. 72
    out = Generator(model, 2, repetition=1.2, presence=50.0, mask=(words.cuda(), None)).generate(prompts, 4)
    assert len(set(out[0])) == 4                 # a token that was said loses 50
    assert sorted(out[1]) == [69, 70, 71, 72]
    again = Generator(model, 2, repetition=1.2, presence=50.0, mask=(words.cuda(), None)).generate(prompts, 4)
    assert out == again
    bias = (torch.tensor([42, 42], dtype=torch.int32, device="cuda"), torch.tensor([60.0, 60.0], device="cuda"),
            torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda"))
    out = Generator(model, 2, bias=bias).generate(prompts, 2)
    assert out[0] == [42, 42]
    with pytest.raises(ValueError):
        Generator(model, 1).forward([[0] * 33])
    with pytest.raises(ValueError):
        Generator(model, 1).forward([[]])
