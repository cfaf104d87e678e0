"""A whole decode with drafted trees over paged caches (blocks.TreeDecoder) on the GPU: the tokens are
those of a plain 64-bit decoder, one at a time, and of the decoder without drafts."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D, HEADS, D_FF, VOCAB, CONTEXT, FRAMES, LAYERS = 128, 2, 256, 500, 96, 30, 2


def weights(rng):
    m = lambda r, c, s: (rng.standard_normal((r, c)) * s).astype(np.float16)  # noqa: E731
    v = lambda n: (0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    norm = lambda: ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32), v(D))  # noqa: E731
    w = {"embed": m(VOCAB, D, 0.6), "positions": (0.6 * rng.standard_normal((CONTEXT, D))).astype(
        np.float32), "norm": norm(), "layers": []}
    for _ in range(LAYERS):
        lay = {"qkv": m(3 * D, D, 0.12), "self_out": m(D, D, 0.2), "cross_q": m(D, D, 0.12),
               "cross_kv": m(2 * D, D, 0.12), "cross_out": m(D, D, 0.2), "fc1": m(D_FF, D, 0.1),
               "fc2": m(D, D_FF, 0.1), "fc1_b": v(D_FF), "fc2_b": v(D)}
        lay["b"] = {"qkv": v(3 * D), "self_out": v(D), "cross_q": v(D), "cross_kv": v(2 * D),
                    "cross_out": v(D)}
        lay.update({k: norm() for k in ("norm_self", "norm_cross", "norm_ffn")})
        w["layers"].append(lay)
    return w


def plain_logits(w, enc, tokens):
    """Logits after the last of `tokens` in 64 bits, the whole sequence anew."""
    f = np.float64
    ln = lambda x, wb: (x - x.mean(-1, keepdims=True)) / np.sqrt(  # noqa: E731
        x.var(-1, keepdims=True) + 1e-5) * wb[0] + wb[1]
    heads = lambda x: x.reshape(len(x), HEADS, -1).transpose(1, 0, 2)  # noqa: E731

    def attend(q, k, v, causal):
        s = heads(q) @ heads(k).transpose(0, 2, 1) / math.sqrt(D // HEADS)
        if causal:
            s = np.where(np.tril(np.ones(s.shape[1:], bool)), s, -np.inf)
        e = np.exp(s - s.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True) @ heads(v)).transpose(1, 0, 2).reshape(len(q), D)

    x = w["embed"][tokens].astype(f) + w["positions"][:len(tokens)]
    erf = np.vectorize(math.erf)
    for lay in w["layers"]:
        b = lay["b"]
        q, k, v = np.split(ln(x, lay["norm_self"]) @ lay["qkv"].astype(f).T + b["qkv"], 3, 1)
        x = x + attend(q, k, v, True) @ lay["self_out"].astype(f).T + b["self_out"]
        q = ln(x, lay["norm_cross"]) @ lay["cross_q"].astype(f).T + b["cross_q"]
        k, v = np.split(enc @ lay["cross_kv"].astype(f).T + b["cross_kv"], 2, 1)
        x = x + attend(q, k, v, False) @ lay["cross_out"].astype(f).T + b["cross_out"]
        h = ln(x, lay["norm_ffn"]) @ lay["fc1"].astype(f).T + lay["fc1_b"]
        x = x + (0.5 * h * (1 + erf(h / math.sqrt(2)))) @ lay["fc2"].astype(f).T + lay["fc2_b"]
    return ln(x[-1], w["norm"]) @ w["embed"].astype(f).T


def plain_greedy(w, enc, prompt, steps, pen, bias, allowed):
    """Tokens and the margins of their picks (the best edited logit over the next)."""
    said, margins = list(prompt), []
    for _ in range(steps):
        x = plain_logits(w, enc, said)
        for t in set(said):
            c = said.count(t)
            x[t] = (x[t] / pen[0] if x[t] > 0 else x[t] * pen[0]) - pen[2] * c - pen[1]
        for t, v in bias.items():
            x[t] += v
        x[~allowed] = -np.inf
        order = np.argsort(-x)
        margins.append(x[order[0]] - x[order[1]])
        said.append(int(order[0]))
    return said[len(prompt):], margins


def encode(w):
    out = {k: w[k] for k in ("positions", "norm")}
    out["embed"] = w["embed"].tobytes()
    out["layers"] = [{k: v.tobytes() if isinstance(v, np.ndarray) and v.dtype == np.float16 else v
                      for k, v in lay.items()} for lay in w["layers"]]
    return out


def branches(rng, known, width):
    """A tree under the last decided token known[0] that holds the chain known[1:] and wrong
    siblings at every node, some with children."""
    tokens, parents, node = [known[0]], [-1], 0
    for right in known[1:]:
        wrong = [int(t) for t in rng.integers(0, VOCAB, width) if t != right]
        at = len(tokens)
        tokens += wrong[:1] + [right] + wrong[1:]
        parents += [node] * (1 + len(wrong))
        tokens.append(int(rng.integers(0, VOCAB)))
        parents.append(at)
        node = at + 1
    return tokens, parents


def test_drafted_decode(gpu_or_new):
    from wavo_b200 import GGML_F16
    from wavo_b200.blocks import TreeDecoder
    gpu = gpu_or_new
    rng = np.random.default_rng(1)
    w = weights(rng)
    enc = rng.standard_normal((4, FRAMES, D)).astype(np.float32)
    prompts = [[3, 7, 11], [5], [9, 2, 2, 8, 1, 4], [6, 6]]
    pen, bias = (1.15, 0.3, 0.1), {17: 0.5, 400: -2.0, 33: -np.inf}
    allowed = rng.random(VOCAB) < 0.8
    steps = 24
    want = [plain_greedy(w, e.astype(np.float64), p, steps, pen, bias, allowed)
            for e, p in zip(enc, prompts)]
    p = gpu.pass_()
    dec = TreeDecoder(gpu, GGML_F16, D, HEADS, D_FF, VOCAB, CONTEXT, FRAMES, 4, encode(w), 40,
                      penalties=pen, bias=bias, allowed=allowed)
    dec.record_cross(p, torch.as_tensor(enc).cuda())
    blocks = int(dec.state[1])

    def decode(draft):
        got = [[t] for t in dec.start(p, prompts)]
        turns = 0
        while min(map(len, got)) < steps and turns < 2 * steps:
            trees = [None if len(g) >= steps else draft(b, g) for b, g in enumerate(got)]
            for b, more in enumerate(dec.verify(p, trees)):
                got[b] += more
            turns += 1
        gpu.sync()
        return [g[:steps] for g in got], turns

    plain, turns = decode(lambda b, g: ([g[-1]], [-1]))
    assert turns == steps - 1
    # f16 operands and 64 bits agree where the pick is not close; the rest of a row goes its own way.
    for b, (tokens, margins) in enumerate(want):
        close = next((i for i, m in enumerate(margins) if m < 0.25), steps)
        assert plain[b][:close] == tokens[:close], b
    assert sum(min([i for i, m in enumerate(mm) if m < 0.25] + [steps]) for _, mm in want) > 20
    # Drafts: right chains of one to five tokens among wrong branches; and nothing but wrong ones.
    good, fast = decode(lambda b, g: branches(rng, [g[-1]] + plain[b][len(g):len(g) + 1 + b], 3))
    assert good == plain and fast < turns
    bad, slow = decode(lambda b, g: ([g[-1], 499, 498, 497], [-1, 0, 0, 2]))
    assert bad == plain
    # Everyone done: every block is free again.
    assert dec.verify(p, [None] * 4) == [[]] * 4
    dec.start(p, [[1]] * 4)
    assert int(dec.state[1]) == blocks - 4


def test_decoder_runs_out_of_blocks(gpu_or_new):
    from wavo_b200 import GGML_F16
    from wavo_b200.blocks import TreeDecoder
    rng = np.random.default_rng(2)
    p = gpu_or_new.pass_()
    dec = TreeDecoder(gpu_or_new, GGML_F16, D, HEADS, D_FF, VOCAB, CONTEXT, FRAMES, 2,
                      encode(weights(rng)), 32, blocks=3)
    dec.record_cross(p, torch.zeros(2, FRAMES, D, device="cuda"))
    first = dec.start(p, [[1] * 16, [2] * 16])
    with pytest.raises(RuntimeError, match="1 segments"):
        dec.verify(p, [([t], [-1]) for t in first])
    # The first segment alone goes on where it was.
    assert len(dec.verify(p, [([first[0]], [-1]), None])[0]) == 1


def test_tokens_and_trees_are_checked_before_the_device(gpu_or_new):
    from wavo_b200 import GGML_F16
    from wavo_b200.blocks import TreeDecoder
    p = gpu_or_new.pass_()
    dec = TreeDecoder(gpu_or_new, GGML_F16, D, HEADS, D_FF, VOCAB, CONTEXT, FRAMES, 2,
                      encode(weights(np.random.default_rng(3))), 8)
    dec.record_cross(p, torch.zeros(2, FRAMES, D, device="cuda"))
    one = ([1], [-1])
    for bad in ([([VOCAB], [-1]), one], [([-1], [-1]), one], [([1, 2], [-1]), one], [one],
                [([1] * 9, list(range(-1, 8))), one], [([1, 2], [-1, 1]), one]):
        with pytest.raises(ValueError):
            dec.verify(p, bad)
    assert len(dec.start(p, [[1], [2, 3]])) == 2
    gpu_or_new.sync()


def test_trees_are_checked(gpu_or_new):
    from wavo_b200.blocks import tree_masks
    m, depth = tree_masks([-1, 0, 0, 2])
    assert m[:, 0].tolist() == [1, 3, 5, 13] and depth.tolist() == [0, 1, 1, 2]
    for bad in ([0], [-1, 1], [-1, -1], [-1, 0, 3]):
        with pytest.raises(ValueError):
            tree_masks(bad)


@pytest.fixture(scope="module")
def gpu_or_new():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()
