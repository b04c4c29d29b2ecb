"""vbs_cu_attention_tree where its numbers are stretched: weights far below
a row's largest, positions far apart, keys that are infinite."""
import numpy as np
import pytest

from test_gpu_tree import TOL, Case

pytestmark = pytest.mark.gpu


@pytest.fixture()
def case(vbs, gpu, clean_errors):
    yield lambda **kw: Case(vbs, **kw)
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"


# ---- weights far below the largest -------------------------------------------
# A weight reaches the product as two fp16 halves beside a largest weight of
# 2^10 or more. Below, one key weighs 1 and all others 2^-31 to 2^-33: their
# high halves are 2 to 8 of fp16's smallest steps (2^-24), rounded, their low
# halves nothing. Rounding each by half a step at random leaves a sum of 1500
# of them off by 0.2% (one deviation), and the spread of the weights, denser
# towards the small ones, by a bias of 0.3%: 2% is eight deviations and the
# bias. (Where they are lost, the whole of a part is missing.)
PLANS = [(1, 2, 2, 64, 1, 3000), (5, 4, 2, 128, 1, 5000), (2, 32, 32, 256, 5, 1500), (5, 32, 8, 256, 20, 1500), (40, 4, 2, 128, 1, 3000),
         (33, 32, 8, 96, 5, 1500), (17, 32, 8, 64, 20, 1500)]


@pytest.mark.parametrize("tokens,nqh,nkh,hd,seqs,n_ctx", PLANS)
@pytest.mark.parametrize("where", ["first", "last"])
def test_many_small_weights_beside_a_large_one(case, tokens, nqh, nkh, hd, seqs, n_ctx, where):
    c = case(seqs=seqs, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(n_ctx,), seed=hd + tokens)
    rng = np.random.default_rng(tokens)
    at = 0 if where == "first" else n_ctx - 1
    c.q[...] = 0.0
    c.q[..., 0] = 1.0 / c.scale
    c.q[..., 1] = 2.0 ** -7 / c.scale        # spreads the scores between fp16's steps
    c.k[..., 0] = -np.log(2.0) * rng.uniform(31, 33, c.k.shape[:3])
    c.k[..., 1] = rng.uniform(-1, 1, c.k.shape[:3])
    c.k[:, :, at, :2] = 0.0
    c.v[...] = rng.uniform(0.5, 1.5, c.v.shape)
    c.v[:, :, at] = 0.0                      # the large weight's own part: nothing hides the others'
    got, (want, _) = c.run(), c.want()
    assert 0 < want.max() < 1e-5
    np.testing.assert_allclose(got, want, rtol=0.02, atol=0)


@pytest.mark.parametrize("tokens,nqh,nkh,hd,seqs,n_ctx", PLANS)
@pytest.mark.parametrize("base", [0.0, 3e6])
def test_scores_that_rise_by_the_most_a_reference_takes(case, tokens, nqh, nkh, hd, seqs, n_ctx, base):
    """Every 128 positions weigh 2^15.94 times the ones before: the weights
    stay below fp16's largest number, however the scores round (3e6: to
    steps of a half). The last ones are nearly all that is left."""
    c = case(seqs=seqs, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(n_ctx,), seed=hd)
    c.q[...] = 0.0
    c.q[..., 0] = 100.0 / c.scale
    c.q[..., 1] = 1.0 / c.scale
    c.k[..., 0] = base / 100.0
    c.k[..., 1] = (np.arange(c.M) // 128) * (15.94 * np.log(2.0))
    c.v[...] = np.abs(c.v) + np.float16(0.5)
    got = c.run()
    for i in range(tokens):
        end = n_ctx + i + 1
        first = (end - 1) // 128 * 128
        for h in range(nqh):
            last = c.v[:, h // (nqh // nkh), first:end].astype(np.float64).mean(1)
            # steps of 15.94 +- 0.1 (keys in fp16) +- 1 (products and scores of 3e6): the 128 before weigh
            # 2^-14.8 each, their values up to 12 times the last ones'
            share = 128.0 / (end - first) * 2.0 ** -14.8
            np.testing.assert_allclose(got[:, i, h], last, rtol=share * 12 + 1e-5, atol=0)


# ---- positions far apart ------------------------------------------------------
@pytest.mark.parametrize("tokens,nqh,nkh,hd,kw", [(4, 4, 2, 64, {}), (3, 2, 1, 256, {}), (20, 4, 1, 128, dict(limit=20000, spare=0)),
                                                  (33, 32, 8, 64, dict(seqs=10))])
@pytest.mark.parametrize("window", [2 ** 30 - 1, 2 ** 31 - 1])
def test_windows_over_positions_at_their_limits(case, tokens, nqh, nkh, hd, kw, window):
    """Queries at the lowest and the highest position there is: the distances
    between them pass what a 32-bit subtraction of the window's edge holds."""
    c = case(tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(300,), window=window, pos=0, tree=True, seed=hd, **kw)
    c.q_pos[:, ::2] = -(2 ** 30 - 1)
    c.q_pos[:, 1::2] = 2 ** 30 - 1
    c.check(weights=True)


# ---- keys that are not finite ---------------------------------------------------
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("tokens,nqh,nkh,hd,kw", [(5, 4, 2, 64, {}), (4, 4, 2, 256, {}), (21, 8, 2, 128, {}),
                                                  (21, 4, 1, 128, dict(limit=20000, spare=0)), (33, 32, 8, 96, dict(seqs=10))])
def test_visible_keys_that_are_not_finite(case, bad, cap, tokens, nqh, nkh, hd, kw):
    """A draft's key, one number of it or all, seen by that draft alone: the
    other rows meet the formula as always. Its own rows
    are NaN for a NaN; an infinite key's score depends on how the query
    splits, so theirs may be anything."""
    c = case(tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(300,), cap=cap, tree=True, seed=tokens, **kw)
    c.sees[:] = np.eye(tokens, dtype=bool)
    c.k[:, :, 302, 5] = bad
    c.k[:, :, 303] = bad
    got, (want, _) = c.run(weights=True), c.want()
    others = [i for i in range(tokens) if i not in (2, 3)]
    np.testing.assert_allclose(got[0][:, others], want[:, others], rtol=0, atol=4 * TOL)
    if np.isnan(bad):
        assert np.isnan(got[0][:, 2:4]).all()
    # the weights of the drafts that other rows alone see
    end = 300 + tokens
    alone = [300 + i for i in others]
    assert np.isfinite(got[1][:, :, alone]).all() and (got[1][:, :, end:] == 7.0).all()
