"""The serving operators through the Python front-end: KVCache and its pages,
DecoderBlock.decode against float64 over the cache's own values, token losses
against the dense one, and all of them together, answering token by token."""

import numpy as np
import pytest

import ember_amd as em
import gpu_helpers as G
from ember_amd import capi, nn
from ember_amd.loss import CrossEntropyLoss, TokenLoss
from ember_amd.optim import SGD
from oracle import serving
from serving_helpers import U

pytestmark = pytest.mark.gpu


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def cached_attention(q, k, v, start, count):
    """float64 causal attention of q (B, T, Hq, D) over k, v (B, L, H, D)."""
    B, T, Hq, D = q.shape
    o = np.zeros(q.shape)
    G_ = Hq // k.shape[2]
    for b in range(B):
        for t in range(count[b]):
            n = start[b] + t + 1
            for h in range(Hq):
                s = k[b, :n, h // G_].astype(np.float64) @ q[b, t, h] / np.sqrt(D)
                e = np.exp(s - s.max())
                o[b, t, h] = e @ v[b, :n, h // G_] / e.sum()
    return o


def test_cache_appends_reads_and_attends():
    rng = np.random.default_rng(0)
    B, H, D = 3, 2, 64
    cache = em.KVCache(B, H, D, tokens=100, page_size=16)
    assert cache.nbytes == B * 7 * 16 * H * D * 2 * 17 // 32
    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]
    for T, count in ((20, [20, 3, 0]), (1, None), (1, None), (30, [30, 30, 30]), (1, [1, 0, 1])):
        start = cache.lengths
        k, v, q = normal(rng, B, T, H, D), normal(rng, B, T, H, D), normal(rng, B, T, 2 * H, D)
        G.say(f"KVCache.write T={T} count={count}")
        cache.write(em.Tensor(k), em.Tensor(v), count)
        n = count or [T] * B
        for b in range(B):
            ks[b].append(k[b, :n[b]]), vs[b].append(v[b, :n[b]])
        assert cache.lengths == [s + c for s, c in zip(start, n)]
        rk, rv = (x.to_np() for x in cache.read())
        for b in range(B):
            for got, all_ in ((rk, ks), (rv, vs)):
                ref = serving.values(*serving.quantise(np.concatenate(all_[b])))
                np.testing.assert_array_equal(got[b, :len(ref)], ref.astype(np.float32))
                assert (got[b, len(ref):] == 0).all()
        o, lse = cache.attention(em.Tensor(q))
        # Weights of a few rounding steps each, over rows of size 1 (see check_attention).
        np.testing.assert_allclose(o.to_np(), cached_attention(q, rk, rv, start, n), rtol=0, atol=64 * U)
        assert lse.shape == (B, 2 * H, T)
        assert all(np.isneginf(lse.to_np()[b, :, n[b]:]).all() for b in range(B))


def test_pages_run_out_and_come_back():
    rng = np.random.default_rng(1)
    cache = em.KVCache(2, 1, 32, tokens=64, page_size=16, pages=4)
    rows = lambda T: (em.Tensor(normal(rng, 2, T, 1, 32)), em.Tensor(normal(rng, 2, T, 1, 32)))  # noqa: E731
    cache.write(*rows(17))                       # two pages each
    with pytest.raises(ValueError, match="pages"):
        cache.write(*rows(16))
    assert cache.lengths == [17, 17]
    cache.write(*rows(15))                       # fills them
    with pytest.raises(ValueError, match="pages"):
        cache.write(*rows(1), count=[1, 0])
    kept = cache.read()[0].to_np()[1]
    cache.reset(0)
    assert cache.lengths == [0, 32]
    with pytest.raises(RuntimeError):
        cache.attention(em.Tensor(normal(rng, 2, 1, 1, 32)))
    k, v = rows(32)
    cache.write(k, v, count=[32, 0])
    got = cache.read()[0].to_np()
    np.testing.assert_array_equal(got[1], kept)
    np.testing.assert_array_equal(got[0], serving.values(*serving.quantise(k.to_np()[0])).astype(np.float32))
    with pytest.raises(ValueError, match="room"):
        cache.write(*rows(33))
    cache.reset()
    assert cache.lengths == [0, 0]
    cache.write(*rows(32))


def decode_reference(block, x, start, count, cached, T):
    """The block on x (B*T, d) in float64, its attention over the values read
    back from its cache, and the projected keys and values."""
    w = {n: getattr(block, n).to_np().astype(np.float64) for n in ("w_qkv", "b_qkv", "w_o", "b_o", "w_1", "b_1", "w_2", "b_2")}
    ln = lambda x, n: (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + n.eps) * n.gamma.to_np() + n.beta.to_np()  # noqa: E731
    x = x.astype(np.float64)
    B = len(start)
    qkv = (ln(x, block.ln1) @ w["w_qkv"] + w["b_qkv"]).reshape(B, T, 3, block.h, block.d // block.h)
    o = cached_attention(qkv[:, :, 0], *cached, start, count).reshape(B * T, block.d)
    x2 = x + o @ w["w_o"] + w["b_o"]
    u = ln(x2, block.ln2) @ w["w_1"] + w["b_1"]
    return x2 + 0.5 * u * (1 + np.tanh(0.8 * u)) @ w["w_2"] + w["b_2"], qkv[:, :, 1], qkv[:, :, 2]


@pytest.mark.parametrize("d, heads", [(128, 2), (256, 2), (128, 4)])
def test_decoder_block_decodes(d, heads):
    rng = np.random.default_rng(d + heads)
    em.random.seed(3)
    block = nn.DecoderBlock(d, heads)
    cache = block.make_cache(2, 64, page_size=16)
    for T, count in ((21, [21, 9]), (1, None), (1, None), (3, [3, 0])):
        start, n = cache.lengths, count or [T, T]
        x = normal(rng, 2 * T, d)
        G.say(f"DecoderBlock.decode d={d} heads={heads} T={T}")
        y = block.decode(em.Tensor(x), cache, count).to_np()
        cached = [t.to_np() for t in cache.read()]
        ref, k, v = decode_reference(block, x, start, n, cached, T)
        # Sums of d and 4d products in fp32 of rows of size 1: the bar of the other block tests.
        np.testing.assert_allclose(y, ref, rtol=1e-3, atol=2e-4)
        for got, exact in zip(cached, (k, v)):
            for b in range(2):
                groups = (n[b], heads, d // heads // 32, 32)
                new, want = got[b, start[b]:start[b] + n[b]].reshape(groups), exact[b, :n[b]].reshape(groups)
                # Within a step of the grid at a group's top (2 of 6) of what was projected.
                assert (np.abs(new - want) <= np.abs(want).max(-1, keepdims=True) / 3 + 1e-5).all()


def test_decode_leaves_training_alone():
    rng = np.random.default_rng(5)
    block = nn.DecoderBlock(128, 2)
    x, g = em.Tensor(normal(rng, 2 * 40, 128)), em.Tensor(normal(rng, 2 * 40, 128))
    capi.set_deterministic(True)
    try:
        block(x, 2, 40)
        dx = block.backward(g).to_np()
        grads = [t.to_np() for t in block.gradients()]
        block(x, 2, 40)
        block.decode(em.Tensor(normal(rng, 6, 128)), block.make_cache(2, 10))
        np.testing.assert_array_equal(block.backward(g).to_np(), dx)
        for a, b in zip(block.gradients(), grads):
            np.testing.assert_array_equal(a.to_np(), b)
    finally:
        capi.set_deterministic(False)


def test_token_logprobs_front_end():
    rng = np.random.default_rng(6)
    x = 3 * normal(rng, 2, 5, 300)
    tokens = rng.integers(-1, 301, (2, 5))
    got = em.token_logprobs(em.Tensor(x), tokens, top=7)
    logp, lse, entropy, order, best = serving.token_logprobs(x.reshape(10, 300), tokens.reshape(10), 7)
    assert got.logp.shape == got.entropy.shape == got.lse.shape == (2, 5) and got.top_logp.shape == (2, 5, 7)
    np.testing.assert_array_equal(got.top_tokens, order.reshape(2, 5, 7))
    for a, b in ((got.logp, logp), (got.lse, lse), (got.entropy, entropy), (got.top_logp, best)):
        np.testing.assert_allclose(a.to_np().reshape(b.shape), b, rtol=0, atol=128 * 8 * U)
    assert em.token_logprobs(em.Tensor(x), tokens.tolist()).top_tokens is None


def test_token_loss_is_the_dense_loss():
    rng = np.random.default_rng(7)
    x = 2 * normal(rng, 64, 50)
    tokens = rng.integers(0, 50, 64)
    dense, sparse = CrossEntropyLoss(), TokenLoss()
    a = dense(em.Tensor(x), em.Tensor(np.eye(50, dtype=np.float32)[tokens]))
    b = sparse(em.Tensor(x), tokens)
    assert abs(a - b) <= 128 * U * abs(a)
    np.testing.assert_allclose(sparse.backward().to_np(), dense.backward().to_np(), rtol=0, atol=32 * U / 64)


def test_token_loss_padded_and_with_entropy():
    rng = np.random.default_rng(8)
    x = 2 * normal(rng, 12, 40)
    tokens = rng.integers(0, 40, 12)
    tokens[[2, 9]] = -1
    known = tokens >= 0
    x[2] = np.nan                               # a padded place holds anything
    loss = TokenLoss(entropy_bonus=0.3)
    value = loss(em.Tensor(x), tokens)
    logp, _, entropy, _, _ = serving.token_logprobs(x[known], tokens[known], 1)
    assert abs(value - (-logp.mean() - 0.3 * entropy.mean())) <= 128 * 8 * U
    grad = loss.backward().to_np()
    n = known.sum()
    ref = serving.token_logprobs_bwd(x[known], tokens[known], np.full(n, -1 / n), np.full(n, -0.3 / n))
    np.testing.assert_allclose(grad[known], ref, rtol=0, atol=64 * U / n)
    assert (grad[~known] == 0).all()
    first = loss.backward()
    first *= 0.0
    np.testing.assert_array_equal(loss.backward().to_np(), grad)
    nothing = TokenLoss()
    assert nothing(em.Tensor(x), np.full(12, -1)) == 0 and (nothing.backward().to_np() == 0).all()


def test_a_head_trains_on_token_ids():
    """Linear and TokenLoss give the parameters the gradients that the dense loss gives."""
    rng = np.random.default_rng(9)
    head = nn.Linear(32, 200)
    x, tokens = em.Tensor(normal(rng, 24, 32)), rng.integers(0, 200, 24)
    loss, dense = TokenLoss(), CrossEntropyLoss()
    y = head(x)
    loss(y, tokens)
    head.backward(loss.backward())
    sparse = [g.to_np() for g in head.gradients()]
    dense(y, em.Tensor(np.eye(200, dtype=np.float32)[tokens]))
    head.backward(dense.backward())
    for a, b in zip(sparse, head.gradients()):
        np.testing.assert_allclose(a, b.to_np(), rtol=0, atol=1e-6)
    SGD(head.parameters(), lr=0.1).apply(head.gradients())


def test_answering_token_by_token():
    """Two blocks with caches and a head: a padded batch of prompts, then the likeliest
    token again and again.  Each step's scores agree with those of the whole text so
    far read at once into fresh caches (as near as their rounded caches are equal)."""
    rng = np.random.default_rng(10)
    em.random.seed(11)
    d, classes, B, P = 128, 300, 2, 18
    blocks = [nn.DecoderBlock(d, 2) for _ in range(2)]
    head = nn.Linear(d, classes)
    table = normal(rng, classes, d)
    lengths = np.array([18, 11])
    text = [list(rng.integers(0, classes, n)) for n in lengths]

    def step(caches, tokens, count=None):
        """tokens (B, T) -> logits of each sequence's last valid row."""
        T = tokens.shape[1]
        x = em.Tensor(table[tokens].reshape(B * T, d))
        for block, cache in zip(blocks, caches):
            x = block.decode(x, cache, count)
        y = x.to_np().reshape(B, T, d)
        last = np.full(B, T) if count is None else np.asarray(count)
        return head(em.Tensor(y[np.arange(B), last - 1]), training=False)

    def padded():
        T = max(len(t) for t in text)
        return np.array([t + [0] * (T - len(t)) for t in text]), [len(t) for t in text]

    def fresh():
        return [b.make_cache(B, 64, page_size=16) for b in blocks]

    caches = fresh()
    logits = step(caches, *padded())
    for i in range(6):
        G.say(f"answer step {i}")
        got = em.token_logprobs(logits, logits.to_np().argmax(-1), top=3)
        best = got.top_tokens[:, 0]
        np.testing.assert_array_equal(best, logits.to_np().argmax(-1))
        np.testing.assert_array_equal(got.logp.to_np(), got.top_logp.to_np()[:, 0])
        assert (got.entropy.to_np() >= 0).all() and (got.entropy.to_np() <= np.log(classes) * (1 + 8 * U)).all()
        for t, token in zip(text, best):
            t.append(int(token))
        logits = step(caches, best[:, None])
        assert caches[0].lengths == [len(t) for t in text]
        again = fresh()
        whole = step(again, *padded())
        same = [a == b for a, b in zip((c.read()[0].to_np().tobytes() for c in caches), (c.read()[0].to_np().tobytes() for c in again))]
        if all(same):
            np.testing.assert_allclose(logits.to_np(), whole.to_np(), rtol=1e-3, atol=2e-4)
        else:  # a projection's last bit turned a code: one step of the grid in one element
            assert np.abs(logits.to_np() - whole.to_np()).max() <= 0.1 * np.abs(whole.to_np()).max()


def test_token_loss_of_more_rows_than_one_grid_takes():
    """2^24 rows and one: every row's gradient, (p - one-hot) / rows."""
    rows = (1 << 24) + 1
    pred = np.zeros((rows, 2), np.float32)
    loss = TokenLoss()
    G.say(f"TokenLoss of {rows} rows")
    assert abs(loss.forward(em.Tensor(pred), np.arange(rows) % 2) - np.log(2)) <= 256 * U  # a sum of 2^24 terms
    got = loss.backward().to_np()
    want = np.where(np.arange(2) == (np.arange(rows) % 2)[:, None], -0.5, 0.5) / rows
    assert (np.abs(got - want) <= 8 * U / rows).all()


@pytest.mark.parametrize("offset", [0.0, -1000.0, 3e4, 1e6])
@pytest.mark.parametrize("bonus", [0.0, 0.3])
def test_token_loss_of_logits_far_from_zero(offset, bonus):
    """Logits with an offset as those without: x - lse is exact where p is not tiny,
    so p is off by the steps of ln s and exp, 16 and 2 |ln p| half steps at most."""
    rng = np.random.default_rng(11)
    rows, classes = 40, 5000
    x = (3 * normal(rng, rows, classes) + np.float32(offset)).astype(np.float32)
    tokens = rng.integers(0, classes, rows)
    loss = TokenLoss(entropy_bonus=bonus)
    loss.forward(em.Tensor(x), tokens)
    grad = loss.backward().to_np()
    m = x.max(-1, keepdims=True).astype(np.float64)
    logp = x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))
    p, entropy = np.exp(logp), -(np.exp(logp) * logp).sum(-1, keepdims=True)
    hot = np.eye(classes)[tokens]
    want = (p - hot + bonus * p * (logp + entropy)) / rows
    size = p + hot + bonus * p * (np.abs(logp) + entropy)
    assert (np.abs(grad - want) <= U * (16 + 4 * np.abs(logp)) * size / rows).all()
    if not bonus:
        dense = CrossEntropyLoss()
        dense.forward(em.Tensor(x), em.Tensor(hot.astype(np.float32)))
        assert (np.abs(dense.backward().to_np() - want) <= U * (32 + 4 * np.abs(logp)) * size / rows).all()
