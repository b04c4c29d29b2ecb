"""vbs_cu_attention_tree against the formula in 64 bits."""
import numpy as np
import pytest

import cache_ops as ref

pytestmark = pytest.mark.gpu

# fp32 arithmetic on halves that carry 22 bits: a score of size |x| is off by
# about |x| 2^-21 (two products of 2^-22, and hd fp32 additions whose errors
# add like their square root), a weight by as much relatively, ex2 by 2^-22.
# Scores here stay below 20: 20 * 2^-21 = 1e-5 per weight at worst, averaged
# over the keys of a row. 2e-5 of the largest value in reach bounds the sum.
TOL = 2e-5


class Case:
    """Inputs of one call in numpy and on the device."""

    def __init__(self, vbs, seqs=1, tokens=1, nqh=8, nkh=2, hd=64, n_ctx=(100,), n_tok=None, head_major=False, layers=1,
                 layer=0, tree=False, cap=0.0, window=0, slopes=False, k_pos=None, pos=None, seed=0, spare=5, qscale=1.0,
                 limit=None):
        import torch
        self.vbs, self.torch = vbs, torch
        rng = np.random.default_rng(seed)
        self.S, self.T, self.nqh, self.H, self.hd, self.cap, self.window = seqs, tokens, nqh, nkh, hd, cap, window
        self.n_ctx = np.asarray([n_ctx[b % len(n_ctx)] for b in range(seqs)])
        self.n_tok = np.full(seqs, tokens) if n_tok is None else np.asarray(n_tok)
        self.limit = limit or max(1, int((self.n_ctx + self.n_tok).max()))
        self.M = self.limit + spare
        self.layers, self.layer, self.head_major = layers, layer, head_major
        self.k = rng.standard_normal((seqs, nkh, self.M, hd)).astype(np.float16)
        self.v = rng.standard_normal((seqs, nkh, self.M, hd)).astype(np.float16)
        self.q = (rng.standard_normal((seqs, tokens, nqh, hd)) * qscale).astype(np.float32)
        self.sees = self.mask = None
        depth = np.tile(np.arange(tokens), (seqs, 1))
        if tree:
            trees = [ref.tree_mask(rng, tokens) for _ in range(seqs)]
            self.sees = np.stack([t[0] for t in trees])
            depth = np.stack([t[1] for t in trees])
        self.q_pos = None if pos is None else (self.n_ctx[:, None] + depth + pos)
        self.k_pos = None if k_pos is None else k_pos(rng, self)
        self.slopes = (2.0 ** (-8.0 * np.arange(1, nqh + 1) / nqh)).astype(np.float32) if slopes else None
        self.scale = 1.0 / np.sqrt(hd)
        self.w_in = rng.random((seqs, nkh, self.M)).astype(np.float32)
        self.stream = 0

    def put(self, a, dtype=None):
        if a is None:
            return None
        return self.torch.from_numpy(np.ascontiguousarray(a if dtype is None else a.astype(dtype))).cuda()

    def cache(self, x):
        """The layer's rows among other layers' NaN, in the case's order."""
        full = np.full((self.S, self.layers) + x.shape[1:], np.nan, dtype=np.float16)
        full[:, self.layer] = x
        if not self.head_major:
            full = full.transpose(0, 1, 3, 2, 4)
        return self.put(full)

    def run(self, weights=False, fill=7.0):
        vbs, put = self.vbs, self.put
        k, v, q = self.cache(self.k), self.cache(self.v), put(self.q)
        out = self.torch.full(self.q.shape, fill, dtype=self.torch.float32, device="cuda")
        keep = [put(self.n_ctx, np.int32), put(self.n_tok, np.int32), put(self.q_pos, np.int32), put(self.k_pos, np.int32),
                put(self.slopes), put(ref.mask_words(self.sees).view(np.int32)) if self.sees is not None else None]
        ptr = [t.data_ptr() if t is not None else None for t in keep]
        w_in, w_out = put(self.w_in), self.torch.full(self.w_in.shape, fill, device="cuda")
        self.kv = vbs.KvDesc(k=k.data_ptr(), v=v.data_ptr(), n_layers=self.layers, max_ctx=self.M, n_kv_heads=self.H,
                             head_dim=self.hd, n_seqs=self.S, head_major=int(self.head_major),
                             seq_stride=self.layers * self.M * self.H * self.hd)
        self.tree = vbs.TreeDesc(n_q_heads=self.nqh, n_tokens=self.T, scale=self.scale, softcap=self.cap, window=self.window,
                                 ctx_limit=self.limit, n_ctx=ptr[0], n_tok=ptr[1], q_pos=ptr[2], k_pos=ptr[3], slopes=ptr[4],
                                 mask=ptr[5], k_pos_per_head=int(self.k_pos is not None and self.k_pos.ndim == 3),
                                 weights_in=w_in.data_ptr() if weights else None,
                                 weights_out=w_out.data_ptr() if weights else None)
        nbytes = vbs.tree_workspace(self.kv, self.tree)
        work = self.torch.full((nbytes,), 255, dtype=self.torch.uint8, device="cuda")   # NaN wherever it is read as float
        self.torch.cuda.synchronize()
        vbs.attention_tree(self.kv, self.layer, self.tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), nbytes, self.stream)
        self.torch.cuda.synchronize()
        return (out.cpu().numpy(), w_out.cpu().numpy()) if weights else out.cpu().numpy()

    def want(self):
        return ref.attend(self.q, self.k, self.v, self.n_ctx, self.n_tok, self.scale, self.sees, self.cap, self.window,
                          self.slopes, self.q_pos, self.k_pos)

    def check(self, weights=False, fill=7.0):
        got = self.run(weights, fill)
        out = got[0] if weights else got
        want, wts = self.want()
        for b in range(self.S):
            t = self.n_tok[b]
            np.testing.assert_allclose(out[b, :t], want[b, :t], rtol=0, atol=TOL * 4)   # values reach about 4
            assert (out[b, t:] == fill).all()      # rows behind the last token: as they were
            if weights:
                end = self.n_ctx[b] + t
                # a sum of T * G weights, each at most 1
                np.testing.assert_allclose(got[1][b, :, :end], (self.w_in + wts)[b, :, :end], rtol=1e-6,
                                           atol=TOL * t * self.nqh / self.H)
                assert (got[1][b, :, end:] == fill).all()
        return out


@pytest.fixture()
def case(vbs, gpu, clean_errors):
    yield lambda **kw: Case(vbs, **kw)
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"


@pytest.mark.parametrize("n_ctx", [0, 1, 15, 16, 63, 64, 65, 127, 1000, 5000])
@pytest.mark.parametrize("head_major", [False, True])
def test_one_token(case, n_ctx, head_major):
    case(n_ctx=(n_ctx,), head_major=head_major, seed=n_ctx).check()


@pytest.mark.parametrize("hd", [8, 32, 64, 80, 96, 112, 128, 200, 256])
@pytest.mark.parametrize("tokens,nqh,nkh", [(1, 3, 3), (5, 8, 2), (9, 6, 2), (17, 8, 1)])
def test_head_dims_and_groups(case, hd, tokens, nqh, nkh):
    case(tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(333,), tree=True, layers=2, layer=1, seed=hd).check()


@pytest.mark.parametrize("tokens", [2, 31, 32, 33, 63, 64, 65, 130])
@pytest.mark.parametrize("tree", [False, True])
def test_tokens(case, tokens, tree):
    case(tokens=tokens, nqh=4, nkh=2, hd=128, n_ctx=(200,), tree=tree, head_major=tree, seed=tokens).check()


@pytest.mark.parametrize("weights", [False, True])
def test_ragged_batch(case, weights):
    case(seqs=6, tokens=7, nqh=8, nkh=4, hd=64, n_ctx=(0, 900, 17, 3000, 64, 1), n_tok=[7, 1, 0, 4, 7, 2], tree=True,
         seed=3).check(weights)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
@pytest.mark.parametrize("n_ctx", [3, 300, 2500])
def test_window(case, window, n_ctx):
    case(seqs=2, tokens=6, nqh=4, nkh=2, hd=64, n_ctx=(n_ctx, n_ctx // 2), window=window, tree=True, pos=0, seed=window).check()
    case(seqs=2, tokens=6, nqh=4, nkh=2, hd=64, n_ctx=(n_ctx, n_ctx // 2), window=window, seed=window).check(weights=True)


@pytest.mark.parametrize("cap,slopes,qscale", [(30.0, False, 4.0), (5.0, False, 10.0), (0.0, True, 1.0), (50.0, True, 3.0)])
def test_cap_and_bias(case, cap, slopes, qscale):
    case(tokens=9, nqh=8, nkh=2, hd=128, n_ctx=(1500,), cap=cap, slopes=slopes, qscale=qscale, tree=True, pos=0, seed=11).check()


def padded(rng, c):
    pad = rng.integers(0, 40, c.S)[:, None]
    kp = np.arange(c.M)[None] - pad
    for b in range(c.S):
        n, t = c.n_ctx[b], c.n_tok[b]
        kp[b, n:n + t] = c.q_pos[b, :t]
    return np.where(kp < 0, -1, kp)


def evicted(rng, c):
    kp = np.cumsum(rng.integers(1, 5, (c.S, c.H, c.M)), -1)
    kp[rng.random(kp.shape) < 0.1] = -1
    for b in range(c.S):
        n, t = c.n_ctx[b], c.n_tok[b]
        kp[b, :, n:n + t] = c.q_pos[b, :t]
    return kp


@pytest.mark.parametrize("k_pos", [padded, evicted])
@pytest.mark.parametrize("window,slopes", [(0, False), (150, False), (0, True)])
def test_positions_of_slots(case, k_pos, window, slopes):
    c = case(seqs=3, tokens=5, nqh=4, nkh=2, hd=64, n_ctx=(400, 90, 700), k_pos=k_pos, pos=700, window=window, slopes=slopes,
             tree=True, head_major=True, seed=21)
    c.check(weights=True)


def test_rows_that_see_nothing_are_zero(case):
    c = case(tokens=4, nqh=4, nkh=2, hd=64, n_ctx=(0,), tree=True, seed=1)
    c.sees[0, 1] = False
    c.sees[0, 3] = False
    out = c.check(weights=True)
    assert (out[0, [1, 3]] == 0).all()
    # everything a hole, over several parts of the positions
    c = case(tokens=2, nqh=2, nkh=1, hd=128, n_ctx=(3000,), k_pos=lambda rng, c: np.full((1, c.M), -1), pos=0, seed=2)
    out = c.check(weights=True)
    assert (out == 0).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_masked_places_may_hold_anything(case, bad):
    """Slots behind the end, holes, drafts of other branches and keys outside
    the window hold infinities or NaN; the rows that do not see them do not
    notice, and the formula (which never reads them) is met."""
    c = case(seqs=2, tokens=6, nqh=4, nkh=2, hd=64, n_ctx=(200, 3), pos=0, tree=True, window=64,
             k_pos=lambda rng, c: padded(rng, c), seed=5)
    c.sees[:, :, 2] = False
    for x in (c.k, c.v):
        for b in range(2):
            end = c.n_ctx[b] + c.n_tok[b]
            x[b, :, end:] = bad
            x[b, :, c.n_ctx[b] + 2] = bad
            x[b, :, :end][:, c.k_pos[b, :end] < 0] = bad
            far = c.q_pos[b].min() - c.k_pos[b, :end] >= 64
            x[b, :, :end][:, far] = bad
    c.check(weights=True)
    # without positions of slots: a window that some rows leave earlier than others
    c = case(tokens=8, nqh=4, nkh=2, hd=128, n_ctx=(100,), window=10, seed=6)
    c.v[0, :, 91:95] = bad   # the first token sees 91.., the fifth 95..
    got, (want, _) = c.run(), c.want()
    assert np.isnan(want[0, :4]).any() or np.isinf(want[0, :4]).any()
    np.testing.assert_allclose(got[0, 4:], want[0, 4:], rtol=0, atol=4 * TOL)
    assert not np.isfinite(got[0, :4]).any()


def test_visible_nan_reaches_its_rows_only(case):
    c = case(tokens=3, nqh=2, nkh=1, hd=64, n_ctx=(4000,), tree=True, seed=8)
    c.sees[0] = np.eye(3, dtype=bool)
    c.k[0, 0, 4001] = np.nan   # the second draft's key, seen by itself alone
    got, (want, _) = c.run(), c.want()
    assert np.isnan(got[0, 1]).all()
    np.testing.assert_allclose(got[0, [0, 2]], want[0, [0, 2]], rtol=0, atol=4 * TOL)
    c.q[0, 2] = np.nan
    got = c.run()
    assert np.isnan(got[0, 2]).all() and np.isfinite(got[0, 0]).all()


@pytest.mark.parametrize("qscale", [1e-30, 1e-4, 1e4])
def test_large_and_small_queries(case, qscale):
    c = case(tokens=2, nqh=4, nkh=2, hd=128, n_ctx=(500,), qscale=qscale, seed=9)
    if qscale > 1:
        c.scale /= qscale
    c.check()


def test_long_context_one_head(case):
    case(tokens=3, nqh=2, nkh=1, hd=64, n_ctx=(70001,), head_major=True, seed=10).check(weights=True)


def test_limit_above_the_lengths(case):
    """ctx_limit is a bound: the same rows with a far larger one."""
    a = case(seqs=2, tokens=3, nqh=8, nkh=2, hd=64, n_ctx=(70, 5), seed=12)
    b = case(seqs=2, tokens=3, nqh=8, nkh=2, hd=64, n_ctx=(70, 5), seed=12, limit=9000, spare=0)
    b.q = a.q
    b.k[:, :, : a.M], b.v[:, :, : a.M] = a.k, a.v
    a.check()
    b.check()


def test_equal_calls_give_equal_bits(case):
    c = case(seqs=3, tokens=20, nqh=16, nkh=2, hd=128, n_ctx=(2500, 31, 700), tree=True, seed=13)
    a, b = c.run(weights=True), c.run(weights=True)
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


def test_bad_lengths_are_reported_and_write_nothing(vbs, gpu, clean_errors):
    for n_ctx, n_tok in (((-1,), [2]), ((50,), [3]), ((60,), [2]), ((50,), [-1])):
        c = Case(vbs, tokens=2, n_ctx=(50,), seed=14, limit=55)
        c.n_ctx, c.n_tok = np.asarray(n_ctx), np.asarray(n_tok)
        out, w = c.run(weights=True)
        assert (out == 7.0).all() and (w == 7.0).all()
        gpu.synchronize_device(gpu.get_device(0))
        assert "invalid data" in vbs.last_error()
        vbs.clear_error()


def test_agrees_with_the_decode_attention(vbs, gpu, clean_errors):
    """One token per sequence over all positions is vbs_cu_attention."""
    import torch
    c = Case(vbs, seqs=2, tokens=1, nqh=32, nkh=8, hd=128, n_ctx=(1233,), seed=15)
    got = c.run()
    k, v, q = c.cache(c.k), c.cache(c.v), c.put(c.q)
    out = torch.empty(c.q.shape, dtype=torch.float32, device="cuda")
    vbs.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1234, 0, c.M, 32, 8, 128, float(c.scale), batch=2,
                  kv_batch_stride=c.M * 8 * 128)
    torch.cuda.synchronize()
    np.testing.assert_allclose(got, out.cpu().numpy(), rtol=0, atol=4 * TOL)


def test_streams_and_graph(vbs, gpu, clean_errors):
    """Captured once, replayed after the lengths changed on the device."""
    import torch
    c = Case(vbs, seqs=2, tokens=4, nqh=8, nkh=2, hd=64, n_ctx=(900, 300), seed=16)
    k, v, q = c.cache(c.k), c.cache(c.v), c.put(c.q)
    out = torch.zeros(c.q.shape, device="cuda")
    n_ctx, n_tok = c.put(c.n_ctx, np.int32), c.put(c.n_tok, np.int32)
    kv = vbs.KvDesc(k=k.data_ptr(), v=v.data_ptr(), n_layers=1, max_ctx=c.M, n_kv_heads=2, head_dim=64, n_seqs=2,
                    head_major=0, seq_stride=c.M * 2 * 64)
    tree = vbs.TreeDesc(n_q_heads=8, n_tokens=4, scale=c.scale, ctx_limit=c.limit, n_ctx=n_ctx.data_ptr(), n_tok=n_tok.data_ptr())
    work = torch.empty(vbs.tree_workspace(kv, tree), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            vbs.attention_tree(kv, 0, tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(), side.cuda_stream)
    torch.cuda.synchronize()
    for lens in ((900, 300), (20, 899), (0, 64)):
        c.n_ctx = np.asarray(lens)
        n_ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want, _ = c.want()
        np.testing.assert_allclose(out.cpu().numpy(), want, rtol=0, atol=4 * TOL)


# ---- many rows of a KV head (other kernels than few rows) -------------------
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_masked_places_may_hold_anything_many_rows(case, bad, hd):
    c = case(seqs=2, tokens=37, nqh=8, nkh=2, hd=hd, n_ctx=(500, 3), pos=0, tree=True, window=64,
             k_pos=lambda rng, c: padded(rng, c), head_major=hd == 96, seed=5)
    c.sees[:, :, 2] = False
    for x in (c.k, c.v):
        for b in range(2):
            end = c.n_ctx[b] + c.n_tok[b]
            x[b, :, end:] = bad
            x[b, :, c.n_ctx[b] + 2] = bad
            x[b, :, :end][:, c.k_pos[b, :end] < 0] = bad
            far = c.q_pos[b].min() - c.k_pos[b, :end] >= 64
            x[b, :, :end][:, far] = bad
    c.check(weights=True)
    # visible to some rows: theirs turn, the others stay
    c = case(tokens=40, nqh=4, nkh=1, hd=hd, n_ctx=(300,), window=100, seed=6)
    c.v[0, 0, 205:207, 3] = bad    # tokens 0..4 (205) and 0..5 (206) see them
    got, (want, _) = c.run(), c.want()
    turned = ~np.isfinite(want)
    assert turned[0, :6, :, 3].all() and turned.sum() == 6 * 4
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    np.testing.assert_allclose(got[~turned], want[~turned], rtol=0, atol=4 * TOL)


@pytest.mark.parametrize("first", [0, 64, 200])
def test_values_not_finite_in_any_tile(case, first):
    """A value that its rows may see in the first, a middle or the last tile,
    next to drafts that it is hidden from."""
    c = case(tokens=30, nqh=4, nkh=1, hd=128, n_ctx=(first,), tree=True, seed=first)
    c.sees[0] = np.eye(30, dtype=bool)
    c.sees[0, :, 0] = True
    c.v[0, 0, first + 7, 11] = np.inf
    c.v[0, 0, first + 9] = np.nan
    got, (want, _) = c.run(), c.want()
    fine = np.isfinite(want)
    assert (~fine).sum() == 4 + 4 * 128 and (got[0, 7, :, 11] == np.inf).all() and np.isnan(got[0, 9]).all()
    np.testing.assert_allclose(got[fine], want[fine], rtol=0, atol=4 * TOL)


@pytest.mark.parametrize("hd", [8, 24, 64, 72, 80, 128])
@pytest.mark.parametrize("n_ctx,tokens", [(0, 5), (0, 130), (90, 33), (127, 1), (128, 64), (1000, 100), (4000, 17)])
def test_many_rows(case, hd, n_ctx, tokens):
    case(seqs=2, tokens=tokens, nqh=40, nkh=2, hd=hd, n_ctx=(n_ctx, n_ctx // 3), tree=True, head_major=hd % 3 == 0,
         layers=2, layer=1, seed=hd + tokens).check()


@pytest.mark.parametrize("cap,slopes,window,qscale", [(30.0, False, 0, 4.0), (0.0, True, 0, 1.0), (5.0, True, 333, 6.0)])
@pytest.mark.parametrize("k_pos", [None, padded, evicted])
def test_many_rows_options(case, cap, slopes, window, qscale, k_pos):
    case(seqs=2, tokens=21, nqh=16, nkh=2, hd=128, n_ctx=(900, 1700), cap=cap, slopes=slopes, window=window, qscale=qscale,
         tree=True, pos=0 if k_pos is None else 1700, k_pos=k_pos, seed=31).check(weights=True)


def test_negative_scale_and_large_scores(case):
    c = case(tokens=20, nqh=4, nkh=1, hd=128, n_ctx=(700,), seed=32)
    c.scale = -c.scale
    c.check()
    c = case(tokens=3, nqh=4, nkh=1, hd=128, n_ctx=(700,), seed=33)
    c.scale = -c.scale
    c.check()


def test_a_late_maximum_moves_the_reference(case):
    """Scores that rise tile by tile, far beyond the lazy threshold."""
    for tokens in (1, 20):
        c = case(tokens=tokens, nqh=4, nkh=1, hd=64, n_ctx=(1500,), seed=34)
        ramp = np.linspace(0, 40, c.M)
        c.q[..., 0] = 1.0 / c.scale
        c.k[0, 0, :, 0] = ramp.astype(np.float16)
        c.check()


@pytest.mark.parametrize("tokens,nqh,nkh,hd,seqs,n_ctx", [(16, 8, 2, 128, 3, 9000), (64, 8, 1, 64, 4, 5000), (1, 2, 2, 128, 2, 9000),
                                                          (3, 4, 1, 256, 2, 6000), (40, 32, 8, 96, 8, 2600)])
def test_long_sums_do_not_drift(case, tokens, nqh, nkh, hd, seqs, n_ctx):
    """Thousands of accumulations: the tensor cores cut their accumulators
    towards zero, by up to a unit of the last place (2^-23 of the value) each.
    An accumulator takes 16 of them (8 of 16 positions, two halves) while it
    grows evenly: 16 * 2^-24 = 9.5e-7 of the result, whatever the context's
    length; left to run over 9000 positions it would reach 35 times that. As
    much again for the scores' accumulators (8 of high halves) and for the
    products' and exponentials' 2^-22."""
    c = case(seqs=seqs, tokens=tokens, nqh=nqh, nkh=nkh, hd=hd, n_ctx=(n_ctx,), seed=hd + tokens)
    c.q[..., 0] = 0.0
    c.v[..., :] += np.float16(2.0)          # values of one sign: a cut shows as a bias
    got, (want, _) = c.run(), c.want()
    bias = ((got - want) / want).mean()
    assert abs(bias) < 2 * 16 * 2.0 ** -24 + 2.0 ** -21
    np.testing.assert_allclose(got, want, rtol=0, atol=8 * TOL)


# ---- the tcgen05 kernel on short lengths -------------------------------------
# The kernel is chosen by ctx_limit, not by the lengths: a large limit sends
# more than 16 rows of a KV head (head_dim up to 128) to the tcgen05 kernel
# whatever the sequences hold, in many parts, most of them empty; many
# sequences send them there in few.
FAR = dict(limit=20000, spare=0)


@pytest.mark.parametrize("hd", [8, 24, 64, 72, 80, 128])
@pytest.mark.parametrize("n_ctx,tokens", [(0, 9), (0, 130), (90, 33), (127, 17), (128, 64), (1000, 40)])
def test_far_limit(case, hd, n_ctx, tokens):
    case(tokens=tokens, nqh=4, nkh=2, hd=hd, n_ctx=(n_ctx,), tree=True, head_major=hd % 3 == 0, seed=hd + tokens, **FAR).check()


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("tokens,nqh", [(18, 2), (33, 6), (64, 4), (65, 8), (150, 2)])
def test_far_limit_ragged(case, tokens, nqh, weights):
    case(seqs=4, tokens=tokens, nqh=nqh, nkh=2, hd=64, n_ctx=(0, 260, 17, 128), n_tok=[tokens, 1, 0, tokens - 1], tree=True, seed=tokens,
         limit=12000, spare=0).check(weights)


@pytest.mark.parametrize("cap,slopes,window,qscale", [(30.0, False, 0, 4.0), (0.0, True, 0, 1.0), (5.0, True, 100, 6.0), (50.0, True, 0, 1.0)])
@pytest.mark.parametrize("k_pos", [None, padded, evicted])
def test_far_limit_options(case, cap, slopes, window, qscale, k_pos):
    case(seqs=2, tokens=21, nqh=8, nkh=2, hd=128, n_ctx=(300, 600), cap=cap, slopes=slopes, window=window, qscale=qscale, tree=True,
         pos=0 if k_pos is None else 700, k_pos=k_pos, seed=41, limit=12000, spare=0).check(weights=True)


@pytest.mark.parametrize("window", [1, 60, 129, 700])
@pytest.mark.parametrize("tree", [False, True])
def test_many_sequences_window(case, window, tree):
    """Few parts: a window's edge inside tiles, its first tile behind others."""
    case(seqs=20, tokens=24, nqh=16, nkh=8, hd=64, n_ctx=(900, 333, 5), window=window, tree=tree, pos=0 if tree else None, seed=window).check()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd,tokens", [(64, 37), (96, 37), (128, 37), (128, 100)])
def test_far_limit_masked_places(case, bad, hd, tokens):
    c = case(seqs=2, tokens=tokens, nqh=4, nkh=2, hd=hd, n_ctx=(400, 3), pos=0, tree=True, k_pos=lambda rng, c: padded(rng, c),
             head_major=hd == 96, seed=5, limit=12000, spare=0)
    c.sees[:, :, 2] = False
    for x in (c.k, c.v):
        for b in range(2):
            end = c.n_ctx[b] + c.n_tok[b]
            x[b, :, end:] = bad
            x[b, :, c.n_ctx[b] + 2] = bad
            x[b, :, :end][:, c.k_pos[b, :end] < 0] = bad
    c.check(weights=True)
    # visible to some rows of some tiles: theirs turn, the others stay
    c = case(tokens=tokens, nqh=4, nkh=1, hd=hd, n_ctx=(300,), tree=True, seed=6, limit=30000, spare=0)
    c.sees[0] = np.eye(tokens, dtype=bool)
    c.sees[0, :, 0] = True
    c.v[0, 0, 307, 3] = bad                      # one row sees it
    c.v[0, 0, 300 + tokens - 1, hd - 1] = bad    # the last
    got, (want, _) = c.run(), c.want()
    turned = ~np.isfinite(want)
    assert turned.sum() == 2 * 4 and (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    np.testing.assert_allclose(got[~turned], want[~turned], rtol=0, atol=4 * TOL)


def test_far_limit_rows_that_see_nothing(case):
    c = case(tokens=30, nqh=4, nkh=2, hd=128, n_ctx=(0,), tree=True, seed=1, **FAR)
    c.sees[0, 3] = False
    c.sees[0, 20:] = False
    out = c.check(weights=True)
    assert (out[0, 3] == 0).all() and (out[0, 20:] == 0).all()
    c = case(tokens=40, nqh=4, nkh=1, hd=128, n_ctx=(3000,), k_pos=lambda rng, c: np.full((1, c.M), -1), pos=0, seed=2, **FAR)
    out = c.check(weights=True)
    assert (out == 0).all()


def test_far_limit_late_maximum_and_nan(case):
    c = case(tokens=20, nqh=4, nkh=1, hd=64, n_ctx=(1500,), seed=34, **FAR)
    c.q[..., 0] = 1.0 / c.scale
    c.k[0, 0, :, 0] = np.minimum(np.arange(c.M) * (40.0 / 1500), 60).astype(np.float16)
    c.check()
    c = case(tokens=20, nqh=4, nkh=1, hd=64, n_ctx=(700,), seed=35, **FAR)
    c.q[0, 5] = np.nan
    got, (want, _) = c.run(), c.want()
    assert np.isnan(got[0, 5]).all()
    rest = [i for i in range(20) if i != 5]
    np.testing.assert_allclose(got[0, rest], want[0, rest], rtol=0, atol=4 * TOL)


@pytest.mark.parametrize("qscale", [1e-30, 1e4])
def test_far_limit_large_and_small_queries(case, qscale):
    c = case(tokens=10, nqh=4, nkh=2, hd=128, n_ctx=(500,), qscale=qscale, seed=9, **FAR)
    if qscale > 1:
        c.scale /= -qscale
    c.check()


def test_two_streams_at_once(vbs, gpu, clean_errors):
    """Two calls that overlap in time, a workspace each, give what they give
    alone; and a captured pair of calls, replayed."""
    import torch
    cases, alone, held = [], [], []
    for k in range(2):
        c = Case(vbs, seqs=4, tokens=20, nqh=8, nkh=2, hd=128, n_ctx=(3000,), seed=50 + k)
        alone.append(c.run())
        kc, vc, q = c.cache(c.k), c.cache(c.v), c.put(c.q)
        n_ctx, out = c.put(c.n_ctx, np.int32), torch.zeros(c.q.shape, device="cuda")
        kv = vbs.KvDesc(k=kc.data_ptr(), v=vc.data_ptr(), n_layers=1, max_ctx=c.M, n_kv_heads=2, head_dim=128, n_seqs=4, head_major=0,
                        seq_stride=c.M * 2 * 128)
        tree = vbs.TreeDesc(n_q_heads=8, n_tokens=20, scale=c.scale, ctx_limit=c.limit, n_ctx=n_ctx.data_ptr())
        work = torch.empty(vbs.tree_workspace(kv, tree), dtype=torch.uint8, device="cuda")
        held.append((kc, vc, q, n_ctx, out, kv, tree, work))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def both(s0, s1):
        for (kc, vc, q, n_ctx, out, kv, tree, work), s in zip(held, (s0, s1)):
            vbs.attention_tree(kv, 0, tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(), s.cuda_stream)

    for _ in range(20):
        both(*streams)
    torch.cuda.synchronize()
    for h, want in zip(held, alone):
        assert (h[4].cpu().numpy() == want).all()
        h[4].zero_()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        with torch.cuda.graph(g, stream=streams[0]):
            both(streams[0], streams[0])
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for h, want in zip(held, alone):
        assert (h[4].cpu().numpy() == want).all()


# ---- many KV heads: 256 rows a CTA; in one part, in parts of a cluster, in
# parts that a second kernel joins
MANY = [(10, 100), (5, 700), (5, 1500), (10, 3000)]


def many(case, seqs, limit, tokens=33, **kw):
    lengths = (limit - tokens, 0, limit // 2, 5, (limit - tokens) // 128 * 128)
    return case(seqs=seqs, tokens=tokens, nqh=32, nkh=8, n_ctx=lengths, n_tok=[(tokens, tokens, 20, 1, 32)[b % 5] for b in range(seqs)],
                limit=limit, spare=0, **kw)


@pytest.mark.parametrize("hd", [64, 72, 128])
@pytest.mark.parametrize("seqs,limit", MANY)
def test_many_heads(case, hd, seqs, limit):
    many(case, seqs, limit, hd=hd, tree=True, head_major=hd == 72, seed=hd).check(weights=limit < 1000)


@pytest.mark.parametrize("cap,slopes,window,qscale", [(30.0, False, 0, 4.0), (0.0, True, 0, 1.0), (5.0, True, 100, 6.0)])
@pytest.mark.parametrize("k_pos", [None, padded, evicted])
def test_many_heads_options(case, cap, slopes, window, qscale, k_pos):
    many(case, 5, 700, hd=128, tree=True, cap=cap, slopes=slopes, window=window, qscale=qscale, pos=0 if k_pos is None else 700, k_pos=k_pos,
         seed=43).check(weights=True)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("seqs,limit", MANY[:2])
def test_many_heads_masked_places(case, bad, seqs, limit):
    c = many(case, seqs, limit, hd=128, pos=0, tree=True, k_pos=lambda rng, c: padded(rng, c), seed=5)
    c.sees[:, :, 2] = False
    for x in (c.k, c.v):
        for b in range(seqs):
            end = c.n_ctx[b] + c.n_tok[b]
            x[b, :, end:] = bad
            if c.n_tok[b] > 2:
                x[b, :, c.n_ctx[b] + 2] = bad
            x[b, :, :end][:, c.k_pos[b, :end] < 0] = bad
    c.check()


@pytest.mark.parametrize("seqs,tokens,nkh,limit", [(5, 9, 8, 100), (10, 2, 8, 100), (1, 5, 2, 700), (1, 2, 2, 1500), (10, 4, 8, 2000)])
def test_wide_heads(case, seqs, tokens, nkh, limit):
    case(seqs=seqs, tokens=tokens, nqh=4 * nkh, nkh=nkh, hd=256, n_ctx=(limit - tokens, 0, 33), limit=limit, spare=0, tree=True,
         seed=tokens).check(weights=limit < 1000)


@pytest.mark.parametrize("hd,tokens,limit", [(64, 3, 500), (128, 33, 700), (256, 3, 500)])
def test_parts_of_a_cluster_in_a_graph(vbs, gpu, clean_errors, hd, tokens, limit):
    """Parts that join themselves, captured and replayed over new lengths."""
    import torch
    c = Case(vbs, seqs=2, tokens=tokens, nqh=8, nkh=2, hd=hd, n_ctx=(limit - tokens, 17), limit=limit, spare=0, seed=hd)
    first = c.run()
    k, v, q = c.cache(c.k), c.cache(c.v), c.put(c.q)
    out = torch.zeros(c.q.shape, device="cuda")
    n_ctx = c.put(c.n_ctx, np.int32)
    c.kv.k, c.kv.v, c.tree.n_ctx, c.tree.n_tok = k.data_ptr(), v.data_ptr(), n_ctx.data_ptr(), None
    nbytes = vbs.tree_workspace(c.kv, c.tree)
    work = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            vbs.attention_tree(c.kv, 0, c.tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), nbytes,
                               torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), first)
    for lengths in ((0, limit - tokens), (129, 64)):
        c.n_ctx = np.asarray(lengths)
        n_ctx.copy_(c.put(c.n_ctx, np.int32))
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_allclose(out.cpu().numpy(), c.want()[0], rtol=0, atol=4 * TOL)
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("tokens,hd,n_ctx", [(7, 64, 500), (33, 128, 700), (33, 256, 300), (5, 128, 2000)])
def test_queries_behind_the_last_token(case, bad, tokens, hd, n_ctx):
    """A padded batch: what the queries of tokens that are not there hold
    reaches neither the rows nor the weights."""
    c = case(seqs=3, tokens=tokens, nqh=8, nkh=2, hd=hd, n_ctx=(n_ctx, 130, 64), n_tok=[1, tokens - 2, 0], seed=tokens)
    for b in range(3):
        c.q[b, c.n_tok[b]:] = bad
    c.check(weights=True)


@pytest.mark.parametrize("tokens,nqh,nkh", [(2, 4, 2), (5, 2, 1), (16, 1, 1)])
@pytest.mark.parametrize("slow", ["first", "every", "none"])
def test_wide_heads_uneven_blocks(case, tokens, nqh, nkh, slow):
    """Heads of 256, many stages a part, some blocks much slower than others
    (holes with values that are not finite): no warp runs ahead of a stage."""
    def holes(rng, c):
        kp = np.tile(np.arange(c.M), (c.S, 1))
        if slow == "first":
            kp[:, 3] = -1
        elif slow == "every":
            kp[:, 5::128] = -1
        return kp

    c = case(seqs=80, tokens=tokens, nqh=nqh, nkh=nkh, hd=256, n_ctx=(1500 - tokens, 700, 1301), limit=1500, spare=0, pos=0, k_pos=holes, seed=tokens)
    c.v[np.broadcast_to((c.k_pos < 0)[:, None, :], c.v.shape[:3])] = np.inf
    first = c.check()
    for _ in range(20):
        assert np.array_equal(c.run(), first, equal_nan=True)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("tokens,hd,seqs", [(1, 64, 1), (5, 256, 3), (9, 96, 9), (41, 112, 2), (70, 64, 3)])
@pytest.mark.parametrize("cap,slopes,window", [(30.0, False, 0), (50.0, True, 0), (5.0, False, 70), (0.0, True, 70)])
def test_bits_do_not_depend_on_what_nobody_sees(case, weights, tokens, hd, seqs, cap, slopes, window):
    """The same rows over other contents of hidden places, slots behind the
    end and queries behind the last token: the same bits while these are
    finite."""
    c = case(seqs=seqs, tokens=tokens, nqh=10, nkh=2, hd=hd, n_ctx=(380, 77, 200), cap=cap, slopes=slopes, window=window, qscale=2.0, tree=True,
             pos=0, n_tok=[max(1, tokens - b) for b in range(seqs)], k_pos=lambda rng, c: padded(rng, c), seed=tokens)
    runs = []
    for fill in (0.0, 60000.0, np.nan, -3.0):
        for b in range(seqs):
            end = c.n_ctx[b] + c.n_tok[b]
            for x in (c.k, c.v):
                x[b, :, end:] = fill
                x[b, :, :end][:, c.k_pos[b, :end] < 0] = fill
            c.q[b, c.n_tok[b]:] = fill
        runs += [c.run(weights), c.run(weights)]
    for k, r in enumerate(runs[1:], 1):
        for w, (a, b) in enumerate(zip(runs[0] if weights else [runs[0]], r if weights else [r])):
            if k // 2 != 2:
                assert np.array_equal(a, b)
            else:
                # NaN: its block adds the visible values one by one instead of
                # on the tensor cores, in another order of roundings. Both sums
                # are within check()'s bound of the formula, so at most twice
                # that apart.
                np.testing.assert_allclose(a, b, rtol=2e-6 * w, atol=2 * (TOL * tokens * 5 if w else 4 * TOL))
