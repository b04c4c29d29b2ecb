"""vbs_cu_attention_tree: every position a row sees counts once, no other
counts at all, on short and long contexts, over all borders of tiles, parts
and row tiles. A position too few or too many shows, however many there are."""
import numpy as np
import pytest

import cache_ops as ref
from test_gpu_tree import Case, evicted, many, padded

pytestmark = pytest.mark.gpu


@pytest.fixture()
def case(vbs, gpu, clean_errors):
    yield lambda **kw: Case(vbs, **kw)
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"


def visible(c, b, h):
    """[token][position] of sequence b and KV head h."""
    n, t = int(c.n_ctx[b]), int(c.n_tok[b])
    see = np.ones((t, n + t), dtype=bool)
    see[:, n:] = np.tril(np.ones((t, t), dtype=bool)) if c.sees is None else c.sees[b, :t, :t]
    qp = c.q_pos[b][:t] if c.q_pos is not None else n + np.arange(t)
    if c.k_pos is None:
        kp = np.concatenate([np.arange(n), qp])
    else:
        kp = (c.k_pos[b, h] if c.k_pos.ndim == 3 else c.k_pos[b])[:n + t]
        see &= kp >= 0
    if c.window:
        see &= qp[:, None] - kp < c.window
    return see


def counts(c, weights=True):
    """Keys of zeros weigh all positions the same, and values of one and zero
    count them modulo head_dim: a weight is a power of two, the sums are whole
    numbers of it, and a result is rounded twice (1 / sum, times sum; an
    approximate reciprocal included 2^-22). A slot's weights go through
    log2(sum), at most 28 and rounded to 2^-20, and 2^-22 of an exponential:
    2^-18 in all."""
    c.k[...] = 0
    c.v[...] = np.arange(c.M)[:, None] % c.hd == np.arange(c.hd)
    c.w_in[...] = 0
    got = c.run(weights=weights)
    out, wts = got if weights else (got, None)
    G = c.nqh // c.H
    for b in range(c.S):
        t, end = int(c.n_tok[b]), int(c.n_ctx[b] + c.n_tok[b])
        for h in range(c.H):
            see = visible(c, b, h)
            seen = np.maximum(see.sum(1), 1)[:, None]
            hits = np.zeros((t, -(-end // c.hd) * c.hd), dtype=np.int64)
            hits[:, :end] = see
            want = hits.reshape(t, -1, c.hd).sum(1) / seen
            for g in range(G):
                np.testing.assert_allclose(out[b, :t, h * G + g], want, rtol=2.0 ** -20, atol=0)
            if weights:
                np.testing.assert_allclose(wts[b, h, :end], G * (see / seen).sum(0), rtol=2.0 ** -18, atol=0)
                assert (wts[b, h, end:] == 7.0).all()
        assert (out[b, t:] == 7.0).all()


LONG = [dict(tokens=3, nqh=2, nkh=1, hd=64, n_ctx=(70001,), head_major=True), dict(tokens=1, nqh=8, nkh=2, hd=128, n_ctx=(131071,)),
        dict(tokens=40, nqh=2, nkh=1, hd=96, n_ctx=(50000,)), dict(tokens=2, nqh=2, nkh=1, hd=256, n_ctx=(33333,)),
        dict(tokens=24, nqh=2, nkh=1, hd=200, n_ctx=(9001,)), dict(tokens=150, nqh=8, nkh=1, hd=64, n_ctx=(8191,))]


@pytest.mark.parametrize("kw", LONG)
@pytest.mark.parametrize("window", [0, 777])
def test_long_contexts(case, kw, window):
    counts(case(window=window, **kw))


@pytest.mark.parametrize("n_ctx", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 255, 256, 1000, 1023])
@pytest.mark.parametrize("tokens,nqh,nkh,hd", [(1, 3, 3, 64), (7, 8, 2, 128), (5, 4, 1, 256), (33, 4, 1, 256), (42, 6, 2, 80), (129, 4, 2, 128)])
def test_every_border(case, n_ctx, tokens, nqh, nkh, hd):
    counts(case(seqs=2, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(n_ctx, n_ctx // 2 + 3), n_tok=[tokens, max(1, tokens - 1)], tree=True,
                seed=n_ctx))


@pytest.mark.parametrize("limit", [20000, 4000])
@pytest.mark.parametrize("tokens,nqh,nkh,hd", [(9, 4, 2, 64), (64, 4, 2, 128), (65, 4, 1, 72), (20, 4, 2, 256)])
def test_far_limits(case, limit, tokens, nqh, nkh, hd):
    counts(case(seqs=3, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(1300, 0, 64), n_tok=[tokens, tokens - 1, 1], tree=True, limit=limit, spare=0,
                seed=hd))


@pytest.mark.parametrize("k_pos,pos", [(padded, 2000), (evicted, 2000), (None, 0)])
@pytest.mark.parametrize("window", [0, 130, 1000])
@pytest.mark.parametrize("tokens,nqh,nkh,hd", [(3, 4, 2, 64), (33, 8, 2, 128), (12, 8, 2, 256)])
def test_holes_and_windows(case, k_pos, pos, window, tokens, nqh, nkh, hd):
    counts(case(seqs=3, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(700, 1999, 90), k_pos=k_pos, pos=pos, window=window, tree=True, seed=window))


@pytest.mark.parametrize("seqs,limit", [(10, 100), (5, 700), (5, 1500), (10, 3000)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_heads(case, seqs, limit, hd):
    counts(many(case, seqs, limit, hd=hd, tree=True, seed=hd))


def test_prompt_chunks(case):
    counts(case(tokens=1025, nqh=4, nkh=2, hd=64, n_ctx=(515,)))
    counts(case(tokens=700, nqh=8, nkh=2, hd=128, n_ctx=(0,), window=129))
    counts(case(tokens=4096, nqh=1, nkh=1, hd=64, n_ctx=(3,)), weights=False)


@pytest.mark.parametrize("kw", LONG + [dict(seqs=2, tokens=21, nqh=16, nkh=2, hd=128, n_ctx=(900, 1700), tree=True)])
def test_weights_to_their_own_size(case, kw):
    """Random scores: a slot's weights to 2 x 2e-5 of themselves (a score's
    error and that of the row's sum), and each row's add up to one."""
    c = case(seed=5, **kw)
    c.w_in[...] = 0
    got, wts = c.run(weights=True)[1], c.want()[1]
    for b in range(c.S):
        end = int(c.n_ctx[b] + c.n_tok[b])
        np.testing.assert_allclose(got[b, :, :end], wts[b, :, :end], rtol=4e-5, atol=0)
        np.testing.assert_allclose(got[b, :, :end].sum(-1, dtype=np.float64), c.n_tok[b] * c.nqh / c.H, rtol=4e-5)


@pytest.mark.parametrize("hd", [104, 128])
def test_wide_row_tiles_with_few_rows_under_load(case, hd):
    """Row tiles of 256 that hold at most 128 rows in most sequences: three
    stages, whose loads come late beside another stream's copies. The result
    is the same in every run."""
    import torch
    c = many(case, 10, 3000, hd=hd, tree=True, seed=hd)
    c.n_tok = np.minimum(c.n_tok, [33] + [32] * 9)
    first = c.check(weights=True)
    k, v, q = c.cache(c.k), c.cache(c.v), c.put(c.q)
    lists = [c.put(x, np.int32) for x in (c.n_ctx, c.n_tok)] + [c.put(ref.mask_words(c.sees).view(np.int32))]
    kv, tree = c.kv, c.tree
    kv.k, kv.v, tree.n_ctx, tree.n_tok, tree.mask = k.data_ptr(), v.data_ptr(), *[x.data_ptr() for x in lists]
    tree.weights_in = tree.weights_out = None
    nbytes = c.vbs.tree_workspace(kv, tree)
    work = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    side, main, big = torch.cuda.Stream(), torch.cuda.Stream(), torch.empty(1 << 29, dtype=torch.uint8, device="cuda")
    outs = [torch.full(c.q.shape, 7.0, device="cuda") for _ in range(50)]
    torch.cuda.synchronize()
    for out in outs:
        with torch.cuda.stream(side):
            big[: 1 << 28].copy_(big[1 << 28:])
        c.vbs.attention_tree(kv, 0, tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), nbytes, main.cuda_stream)
    torch.cuda.synchronize()
    for out in outs:
        assert np.array_equal(out.cpu().numpy(), first)
