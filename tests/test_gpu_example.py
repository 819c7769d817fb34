"""The calls of the 16-bit layers together (example_kv16: prefill, fork, decode steps over 16-bit and sealed layers, free,
compact) against the same model in plain torch."""
import math

import pytest

import sjk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _rotated(T, ex, m, il, x, pos):
    """q, k, v of rows x at positions pos, in 32 bits from the projection's bf16 rows."""
    import kv16
    q, k, v = (y.float() for y in m.heads(il, x))
    step, _ = kv16.rope_steps(ex.D, base=1e5)
    ang = T.tensor([[(p * s % 2 ** 64) * 2.0 ** -64 * 2 * math.pi for s in step] for p in pos], dtype=T.float64, device="cuda").float()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    out = []
    for y, w in zip((q, k), m.norms[il]):
        y = y * T.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = y[..., : ex.D // 2], y[..., ex.D // 2:]
        out.append(T.cat((a * c - b * s, a * s + b * c), -1))
    return out[0], out[1], v


@pytest.mark.parametrize("kinds,bound", [(("kv16", "kv16"), 0.02), (("kv16", "sealed", "kv16"), 0.06)])
def test_samples_of_a_prompt(T, kinds, bound):
    """Logits of every sample and step against plain attention over the whole history. Bound: the caches' rounding. bf16
    rows and queries are off by up to 2^-8 of a value in each of two layers (K, V and q: under 0.02 of the logits in the
    norm); the sealed layer's tail holds 6-bit rows, off by about 0.03 in the norm (64 centroids)."""
    import example_kv16 as ex
    n, prompt, steps = 3, 77, 25
    m = ex.Model(kinds)
    srv = ex.Server(m, n, prompt + steps + ex.PAGE)
    g = T.Generator(device="cuda")
    g.manual_seed(3)
    tokens = T.randint(0, ex.VOCAB, (prompt,), device="cuda", generator=g)
    forced = T.randint(0, ex.VOCAB, (steps, n), device="cuda", generator=g)
    srv.prefill(tokens)
    used = srv.pages.c.n_pages - srv.pages.n_free.item()
    assert used == -(-prompt // ex.PAGE) and srv.fork(n).tolist() == [0] * (n - 1)
    # plain: K, V of every layer and sample as growing lists
    hist = []
    for il in range(len(kinds)):
        _, k, v = _rotated(T, ex, m, il, m.embed[tokens], range(prompt))
        hist.append([(k, v) for _ in range(n)])
    for i in range(steps):
        got = srv.step(forced[i], prompt + i)
        x = m.embed[forced[i]]
        for il in range(len(kinds)):
            q, k, v = _rotated(T, ex, m, il, x, [prompt + i] * n)
            att = []
            for s in range(n):
                K, V = (T.cat((h, y[s:s + 1])) for h, y in zip(hist[il][s], (k, v)))
                hist[il][s] = K, V
                w = T.softmax(T.einsum("hgd,thd->hgt", q[s].view(ex.HEADS_KV, -1, ex.D), K) / math.sqrt(ex.D), -1)
                att.append(T.einsum("hgt,thd->hgd", w, V).reshape(-1))
            x = x + T.stack(att) @ m.wo[il]
        want = x @ m.embed.T
        err = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
        assert err <= bound, f"step {i}: {err}"
    # the prompt's full pages were shared: every sample added the pages of its own tokens only
    per = -(-(prompt + steps) // ex.PAGE)
    own = per - prompt // ex.PAGE
    used = srv.pages.c.n_pages - srv.pages.n_free.item()
    assert used == prompt // ex.PAGE + n * own
    top, _ = srv.finish(n).tolist()
    assert top == per and sorted(srv.cache.tables[0, :per].tolist()) == list(range(per))
    assert srv.step(forced[0][:1], prompt + steps).shape == (1, ex.VOCAB)
    assert sjk.lib().sjk_device_status() == 0
    srv.close()
