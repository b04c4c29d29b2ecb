"""vbs_cu_rope_store, vbs_cu_cache_select and vbs_cu_cache_gather against
their definitions, and a run of the cache operators together."""
import numpy as np
import pytest

import cache_ops as ref

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype=dtype))).cuda()


def kv_of(vbs, k, v, head_major):
    """KvDesc of [seq][layer][position][head][hd] (or head-major) tensors."""
    S, L, a, b, hd = k.shape
    ctx, heads = (b, a) if head_major else (a, b)
    return vbs.KvDesc(k=k.data_ptr(), v=v.data_ptr(), n_layers=L, max_ctx=ctx, n_kv_heads=heads, head_dim=hd, n_seqs=S,
                      head_major=int(head_major), seq_stride=L * ctx * heads * hd)


@pytest.fixture(autouse=True)
def no_errors(vbs, gpu, clean_errors):
    yield
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"


def device_error(vbs, gpu):
    gpu.synchronize_device(gpu.get_device(0))
    said = vbs.last_error()
    vbs.clear_error()
    return said


# ---- rotary positions ------------------------------------------------------
# Angle: the fraction of a circle to 2^-24 of half a circle, so 2 pi 2^-25 =
# 1.9e-7; sine and cosine of 2^-23; products and sum 3 * 2^-24: below 5e-7 of
# the pair's length, which stays under 6 for standard normals.
ROPE_TOL = 6 * 5e-7


@pytest.mark.parametrize("hd,rot", [(8, 8), (64, 64), (80, 32), (96, 96), (128, 128), (128, 64), (256, 256), (200, 104)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("head_major", [False, True])
def test_rope_store(vbs, hd, rot, halves, head_major):
    import torch
    rng = np.random.default_rng(hd + rot)
    n, nqh, nkh, S, L, ctx = 13, 5, 2, 3, 2, 40
    q, k, v = (rng.standard_normal((n, h, hd)).astype(np.float32) for h in (nqh, nkh, nkh))
    pos = rng.integers(-5, 200000, (n, 1))
    seq = rng.integers(0, S, n)
    slot = rng.permutation(ctx)[:n]
    slot[3] = -1
    shape = (S, L, nkh, ctx, hd) if head_major else (S, L, ctx, nkh, hd)
    kc, vc = (torch.full(shape, 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    plan = vbs.rope_plan(hd, rot_dim=rot, theta=500000.0, halves=halves)
    out = torch.zeros((n, nqh, hd), device="cuda")
    d = [dev(q), dev(k), dev(v), dev(pos, np.int32), dev(slot, np.int32), dev(seq, np.int32)]
    vbs.rope_store(plan, kv_of(vbs, kc, vc, head_major), 1, d[0].data_ptr(), out.data_ptr(), nqh, d[1].data_ptr(),
                   d[2].data_ptr(), n, d[3].data_ptr(), d[4].data_ptr(), seq=d[5].data_ptr())
    torch.cuda.synchronize()
    axis = np.zeros(rot // 2, dtype=np.int64)
    np.testing.assert_allclose(out.cpu().numpy(), ref.rope(q, pos, axis, rot, 500000.0, halves), rtol=0, atol=ROPE_TOL)
    kw = ref.rope(k, pos, axis, rot, 500000.0, halves)
    gk, gv = (x.cpu().numpy() if not head_major else x.cpu().numpy().transpose(0, 1, 3, 2, 4) for x in (kc, vc))
    seen = np.zeros((S, L, ctx), dtype=bool)
    for i in range(n):
        if slot[i] < 0:
            continue
        seen[seq[i], 1, slot[i]] = True
        # half a step of fp16 (2^-11), and the turn's error
        np.testing.assert_allclose(gk[seq[i], 1, slot[i]].astype(np.float64), kw[i], rtol=2.0 ** -11, atol=ROPE_TOL)
        assert (gv[seq[i], 1, slot[i]] == v[i].astype(np.float16)).all()
    assert (gk[~seen] == 7.0).all() and (gv[~seen] == 7.0).all()


@pytest.mark.parametrize("sections,interleaved", [([16, 24, 24], False), ([24, 20, 20], True), ([40, 24], False),
                                                  ([1, 21, 21, 21], True), ([0, 64], False)])
def test_rope_axes(vbs, sections, interleaved):
    import torch
    rng = np.random.default_rng(1)
    n, nqh, hd = 300, 4, 128
    A = len(sections)
    q = rng.standard_normal((n, nqh, hd)).astype(np.float32)
    pos = rng.integers(0, 5000, (n, A))
    fac = 1.0 + 7.0 * rng.random(64)
    axis = np.asarray([p % A if p < A * sections[p % A] else 0 for p in range(64)] if interleaved else
                      [a for a in range(A) for _ in range(sections[a])])
    plan = vbs.rope_plan(hd, halves=True, sections=sections, interleaved=interleaved, freq_factors=list(fac))
    assert list(plan.axis[:64]) == list(axis)
    d = [dev(q), dev(pos, np.int32)]
    vbs.rope_store(plan, None, 0, d[0].data_ptr(), d[0].data_ptr(), nqh, 0, 0, n, d[1].data_ptr(), 0)   # in place, no store
    torch.cuda.synchronize()
    np.testing.assert_allclose(d[0].cpu().numpy(), ref.rope(q, pos, axis, hd, 10000.0, True, fac), rtol=0, atol=ROPE_TOL)


def test_rope_strided_rows_and_store_only(vbs):
    """q | k | v rows of one fused projection; then keys and values alone."""
    import torch
    rng = np.random.default_rng(2)
    n, nqh, nkh, hd, ctx = 9, 6, 2, 64, 16
    x = rng.standard_normal((n, (nqh + 2 * nkh) * hd)).astype(np.float32)
    pos = np.arange(n)[:, None] + 100000
    kc, vc = (torch.zeros((1, 1, ctx, nkh, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    out = torch.zeros((n, nqh, hd), device="cuda")
    d = [dev(x), dev(pos, np.int32), dev(np.arange(n)[::-1] + 2, np.int32)]
    plan, kv = vbs.rope_plan(hd), kv_of(vbs, kc, vc, False)
    row = x.shape[1]
    p = d[0].data_ptr()
    vbs.rope_store(plan, kv, 0, p, out.data_ptr(), nqh, p + nqh * hd * 4, p + (nqh + nkh) * hd * 4, n, d[1].data_ptr(),
                   d[2].data_ptr(), q_stride=row, kv_stride=row)
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    vbs.rope_store(plan, kv_of(vbs, k2, v2, False), 0, 0, 0, 0, p + nqh * hd * 4, p + (nqh + nkh) * hd * 4, n,
                   d[1].data_ptr(), d[2].data_ptr(), kv_stride=row)
    torch.cuda.synchronize()
    axis = np.zeros(hd // 2, dtype=np.int64)
    xs = x.reshape(n, -1, hd)
    np.testing.assert_allclose(out.cpu().numpy(), ref.rope(xs[:, :nqh], pos, axis, hd, 10000.0, False), rtol=0, atol=ROPE_TOL)
    want = ref.rope(xs[:, nqh:nqh + nkh], pos, axis, hd, 10000.0, False)[::-1]
    np.testing.assert_allclose(kc[0, 0, 2:2 + n].cpu().numpy().astype(np.float64), want, rtol=2.0 ** -11, atol=ROPE_TOL)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)


def test_rope_far_positions(vbs):
    """The first pair turns by one radian per position: the whole range of
    positions keeps the tolerance."""
    import torch
    q = np.zeros((5, 1, 64), dtype=np.float32)
    q[..., 0] = 1.0
    pos = np.asarray([[2 ** 31 - 1], [-2 ** 31], [10 ** 9 + 7], [3], [0]])
    d = [dev(q), dev(pos, np.int32)]
    out = torch.zeros((5, 1, 64), device="cuda")
    vbs.rope_store(vbs.rope_plan(64), None, 0, d[0].data_ptr(), out.data_ptr(), 1, 0, 0, 5, d[1].data_ptr(), 0)
    torch.cuda.synchronize()
    ang = pos[:, 0].astype(np.float64)   # exact; the plan's turn is off by 2^-53 of itself, 2^31 positions by 2^-22 of a radian
    got = out.cpu().numpy()[:, 0, :2]
    np.testing.assert_allclose(got, np.stack([np.cos(ang), np.sin(ang)], 1), rtol=0, atol=1e-6)


def test_rope_bad_slots_are_reported(vbs, gpu):
    import torch
    n, hd, ctx = 4, 64, 8
    kc, vc = (torch.full((2, 1, ctx, 1, hd), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    x = torch.ones((n, 1, hd), device="cuda")
    for slot, seq, fine in (([0, 8, -2, 1], [0, 0, 0, 1], [0, 3]), ([0, 1, 2, 3], [0, 2, -1, 1], [0, 3])):
        kc.fill_(7.0)
        d = [dev(slot, np.int32), dev(seq, np.int32), dev(np.zeros(n), np.int32)]
        vbs.rope_store(vbs.rope_plan(hd), kv_of(vbs, kc, vc, False), 0, 0, 0, 0, x.data_ptr(), x.data_ptr(), n, d[2].data_ptr(),
                       d[0].data_ptr(), seq=d[1].data_ptr())
        assert "invalid data" in device_error(vbs, gpu)
        want = torch.full_like(kc, 7.0)
        for i in fine:
            want[seq[i], 0, slot[i]] = 1.0
        assert torch.equal(kc, want)


def test_rope_padding_names_no_sequence(vbs):
    """A token without a slot may carry any sequence number."""
    import torch
    n, hd, ctx = 4, 64, 8
    kc, vc = (torch.full((2, 1, ctx, 1, hd), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    x = torch.ones((n, 1, hd), device="cuda")
    q = torch.zeros_like(x)
    d = [dev([-1, 5, -1, -1], np.int32), dev([-1, 1, 2, 1 << 30], np.int32), dev(np.zeros(n), np.int32)]
    vbs.rope_store(vbs.rope_plan(hd), kv_of(vbs, kc, vc, False), 0, x.data_ptr(), q.data_ptr(), 1, x.data_ptr(), x.data_ptr(), n,
                   d[2].data_ptr(), d[0].data_ptr(), seq=d[1].data_ptr())
    want = torch.full_like(kc, 7.0)
    want[1, 0, 5] = 1.0
    assert torch.equal(kc, want) and torch.equal(vc, want) and torch.equal(q, x)


# ---- selection -------------------------------------------------------------
def scores_of(kind, rng, shape):
    x = np.exp(rng.standard_normal(shape) * 3).astype(np.float32)
    if kind == "ties":
        x = np.round(x).astype(np.float32)
    elif kind == "signs":
        x = (rng.standard_normal(shape) * 1e-3).astype(np.float32)
        x[..., ::7] = 0.0
        x[..., 3::7] = -0.0
    elif kind == "equal":
        x[...] = 2.5
    elif kind == "strange":
        pick = rng.integers(0, 6, shape)
        x = np.select([pick == 0, pick == 1, pick == 2, pick == 3], [np.nan, np.inf, -np.inf, np.float32(1e-44)], x)
    elif kind == "near":   # neighbours in the last bit
        x = (np.float32(1.0) + rng.integers(0, 50, shape) * np.float32(2.0 ** -23)).astype(np.float32)
    return x.astype(np.float32)


def run_select(vbs, x, n, keep, first, recent, limit=None):
    import torch
    L, S, H, stride = x.shape
    idx = torch.full((L, S, H, keep), 77, dtype=torch.int32, device="cuda")
    count = torch.full((S,), 77, dtype=torch.int32, device="cuda")
    d = [dev(x), dev(n, np.int32)]
    vbs.cache_select(d[0].data_ptr(), stride, L, S, H, d[1].data_ptr(), limit or stride, keep, first, recent, idx.data_ptr(),
                     count.data_ptr())
    torch.cuda.synchronize()
    return idx.cpu().numpy(), count.cpu().numpy()


@pytest.mark.parametrize("kind", ["plain", "ties", "signs", "equal", "strange", "near"])
@pytest.mark.parametrize("n,keep,first,recent", [(1, 1, 0, 0), (33, 7, 2, 3), (512, 511, 0, 0), (513, 100, 4, 96), (3000, 1, 1, 0),
                                                 (3000, 1, 0, 0), (5000, 1000, 4, 128), (5000, 4999, 0, 4999)])
def test_select(vbs, kind, n, keep, first, recent):
    rng = np.random.default_rng(n + keep)
    x = scores_of(kind, rng, (2, 2, 3, n + 3))
    idx, count = run_select(vbs, x, [n, max(1, n - 1)], keep, first, recent)
    for s, m in enumerate((n, max(1, n - 1))):
        assert count[s] == min(m, keep)
        for l in range(2):
            for h in range(3):
                assert (idx[l, s, h] == ref.select(x[l, s, h], m, keep, first, recent)).all(), (l, s, h)


@pytest.mark.parametrize("n,keep,lists", [(20000, 3000, 1), (70000, 2048, 1), (131072, 65537, 2), (360448, 5, 1), (3145728, 1000, 1), (60000, 20000, 40)])
def test_select_long(vbs, n, keep, lists):
    rng = np.random.default_rng(n)
    x = scores_of("ties", rng, (1, 1, lists, n))
    idx, _ = run_select(vbs, x, [n], keep, 4, min(keep - 4, 64))
    for h in range(lists):
        assert (idx[0, 0, h] == ref.select(x[0, 0, h], n, keep, 4, min(keep - 4, 64))).all()


@pytest.mark.parametrize("n", [260, 2600])
@pytest.mark.parametrize("share", range(1, 26, 2))
def test_select_border(vbs, n, share):
    """The border falls into every kind of value, its ends and neighbours."""
    kinds = np.asarray([np.nan, np.inf, -np.inf, 1e-44, -1e-44, 0.0, -0.0, 3.4e38, -3.4e38, 1.0, -1.0, 1.1754944e-38, -1.1754944e-38], dtype=np.float32)
    x = kinds[np.random.default_rng(share).integers(0, 13, (1, 1, 2, n))]
    keep = n * share // 26
    idx, _ = run_select(vbs, x, [n], keep, 3, 2)
    for h in range(2):
        assert (idx[0, 0, h] == ref.select(x[0, 0, h], n, keep, 3, 2)).all()


def test_select_short_and_empty(vbs):
    x = scores_of("plain", np.random.default_rng(0), (1, 3, 2, 300))
    idx, count = run_select(vbs, x, [0, 5, 20], 20, 3, 3)
    assert list(count) == [0, 5, 20]
    assert (idx[0, 0] == -1).all() and (idx[0, 1, :, :5] == np.arange(5)).all() and (idx[0, 1, :, 5:] == -1).all()
    assert (idx[0, 2] == np.arange(20)).all()


def test_select_bad_lengths_are_reported(vbs, gpu):
    x = scores_of("plain", np.random.default_rng(0), (1, 3, 2, 100))
    idx, count = run_select(vbs, x, [-1, 101, 100], 20, 3, 3)
    assert "invalid data" in device_error(vbs, gpu)
    assert list(count) == [77, 77, 20] and (idx[0, :2] == 77).all() and (idx[0, 2] >= 0).all()


# ---- row moves -------------------------------------------------------------
@pytest.mark.parametrize("hd", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("sm,dm", [(False, False), (True, True), (False, True)])
def test_gather_apart(vbs, hd, sm, dm):
    import torch
    rng = np.random.default_rng(hd)
    L, S, H, ctx, dctx, n = 2, 3, 2, 90, 61, 50
    rows = rng.standard_normal((2, S, L, H, ctx, hd)).astype(np.float16)
    k, v = (dev(r if sm else r.transpose(0, 1, 3, 2, 4)) for r in rows)
    shape = (S, L, H, dctx, hd) if dm else (S, L, dctx, H, hd)
    k2, v2 = (torch.full(shape, 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    idx = rng.integers(0, ctx - 20, (L, S, H, n))          # any order, repeats
    count, sb, db = np.asarray([n, 0, 13]), np.asarray([20, 0, 5]), np.asarray([11, 3, 0])
    w, p = rng.random((L, S, H, ctx)).astype(np.float32), rng.integers(0, 1000, (L, S, H, ctx)).astype(np.int32)
    d = [dev(a, np.int32) for a in (idx, count, sb, db)] + [dev(w), dev(p)]
    w2, p2 = torch.full((L, S, H, dctx), 7.0, device="cuda"), torch.full((L, S, H, dctx), 7, dtype=torch.int32, device="cuda")
    g = vbs.GatherDesc(n_max=n, idx=d[0].data_ptr(), layer_stride=S * H * n, seq_stride=H * n, head_stride=n,
                       count=d[1].data_ptr(), src_base=d[2].data_ptr(), dst_base=d[3].data_ptr(), weights_src=d[4].data_ptr(),
                       weights_dst=w2.data_ptr(), pos_src=d[5].data_ptr(), pos_dst=p2.data_ptr())
    vbs.cache_gather(kv_of(vbs, k, v, sm), kv_of(vbs, k2, v2, dm), g)
    torch.cuda.synchronize()
    for src, got in zip(rows, (k2, v2)):
        want = np.full((S, L, H, dctx, hd), 7.0, dtype=np.float16)
        for l in range(L):
            for s in range(S):
                for h in range(H):
                    at = idx[l, s, h, : count[s]] + sb[s]
                    want[s, l, h, db[s]:db[s] + count[s]] = src[s, l, h, at]
        got = got.cpu().numpy()
        assert (got == (want if dm else want.transpose(0, 1, 3, 2, 4))).all()
    for src, got in ((w, w2), (p, p2)):
        want = np.full((L, S, H, dctx), 7, dtype=src.dtype)
        for l, s, h in np.ndindex(L, S, H):
            want[l, s, h, db[s]:db[s] + count[s]] = src[l, s, h, idx[l, s, h, : count[s]] + sb[s]]
        assert (got.cpu().numpy() == want).all()


@pytest.mark.parametrize("hd,head_major", [(8, False), (64, True), (80, False), (128, False), (256, True)])
@pytest.mark.parametrize("n,ctx", [(5, 40), (700, 1500), (1500, 1500)])
def test_gather_in_place(vbs, hd, head_major, n, ctx):
    import torch
    rng = np.random.default_rng(hd + n)
    L, S, H = 2, 2, 3
    rows = rng.standard_normal((2, S, L, H, ctx + 9, hd)).astype(np.float16)
    k, v = (dev(r if head_major else r.transpose(0, 1, 3, 2, 4)) for r in rows)
    idx = np.sort(np.stack([rng.permutation(ctx)[:n] for _ in range(L * S * H)]).reshape(L, S, H, n), -1)
    count, sb, db = np.asarray([n, n // 2]), np.asarray([9, 4]), np.asarray([2, 4])
    w = rng.random((L, S, H, ctx + 9)).astype(np.float32)
    d = [dev(a, np.int32) for a in (idx, count, sb, db)] + [dev(w)]
    g = vbs.GatherDesc(n_max=n, idx=d[0].data_ptr(), layer_stride=S * H * n, seq_stride=H * n, head_stride=n,
                       count=d[1].data_ptr(), src_base=d[2].data_ptr(), dst_base=d[3].data_ptr(), weights_src=d[4].data_ptr(),
                       weights_dst=d[4].data_ptr())
    kv = kv_of(vbs, k, v, head_major)
    vbs.cache_gather(kv, kv, g)
    torch.cuda.synchronize()
    for src, got in zip(rows, (k, v)):
        want = src.copy()
        for l, s, h in np.ndindex(L, S, H):
            want[s, l, h, db[s]:db[s] + count[s]] = src[s, l, h, idx[l, s, h, : count[s]] + sb[s]]
        got = got.cpu().numpy()
        assert (got == (want if head_major else want.transpose(0, 1, 3, 2, 4))).all()
    want = w.copy()
    for l, s, h in np.ndindex(L, S, H):
        want[l, s, h, db[s]:db[s] + count[s]] = w[l, s, h, idx[l, s, h, : count[s]] + sb[s]]
    assert (d[4].cpu().numpy() == want).all()


def test_gather_bad_lists_are_reported(vbs, gpu):
    import torch
    k = torch.arange(2 * 30 * 8, device="cuda").reshape(2, 1, 30, 1, 8).half()
    v = k.clone()
    kv = kv_of(vbs, k, v, False)
    k0 = k.clone()
    for lists, count in (([[5, 4, 6], [0, 1, 2]], [3, 3]),      # not ascending
                         ([[5, 5, 6], [0, 1, 2]], [3, 3]),      # the same row twice
                         ([[5, 6, 30], [0, 1, 2]], [3, 3]),     # behind the cache
                         ([[-1, 6, 7], [0, 1, 2]], [3, 3]),     # moves up
                         ([[5, 6, 7], [0, 1, 2]], [4, 3]),      # longer than the lists
                         ([[5, 6, 7], [0, 1, 2]], [-1, 3])):
        d = [dev(lists, np.int32), dev(count, np.int32)]
        g = vbs.GatherDesc(n_max=3, idx=d[0].data_ptr(), seq_stride=3, count=d[1].data_ptr())
        vbs.cache_gather(kv, kv, g)
        assert "invalid data" in device_error(vbs, gpu)
        assert torch.equal(k, k0) and torch.equal(v, k0)
    # apart: the bad row alone stays behind
    k2, v2 = (torch.full((2, 1, 4, 1, 8), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    d = [dev([[29, 30, 3], [-1, 0, 1]], np.int32), dev([3, 3], np.int32)]
    g = vbs.GatherDesc(n_max=3, idx=d[0].data_ptr(), seq_stride=3, count=d[1].data_ptr())
    vbs.cache_gather(kv, kv_of(vbs, k2, v2, False), g)
    assert "invalid data" in device_error(vbs, gpu)
    assert torch.equal(k2[0, 0, :3:2], k[0, 0, [29, 3]]) and (k2[0, 0, 1] == 7).all() and (k2[1, 0, 0] == 7).all()


# ---- together --------------------------------------------------------------
def test_prompt_eviction_and_drafts_together(vbs):
    """A prompt with two position axes goes into a cache; its last tokens'
    attention weights choose what stays; the rows move to a small cache; a
    tree of drafts is attended over it; the accepted branch is moved behind the
    context; the next token attends over what is left. Every step's result
    against the definitions on the device's own inputs."""
    import torch
    rng = np.random.default_rng(5)
    S, nqh, H, hd, L, P, W = 2, 8, 2, 64, 1, 150, 16
    keep, T = 60, 11
    plan = vbs.rope_plan(hd, sections=[20, 12])
    axis = np.asarray(list(plan.axis[: hd // 2]))
    M, M2 = P + 1, keep + T + 2
    kc, vc = (torch.zeros((S, L, M, H, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    k2, v2 = (torch.zeros((S, L, H, M2, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    big, small = kv_of(vbs, kc, vc, False), kv_of(vbs, k2, v2, True)

    def attention(kv, n_ctx, limit, q, q_pos, sees=None, k_pos=None, weights=None):
        t = q.shape[1]
        out = torch.zeros(q.shape, device="cuda")
        hold = [dev(q_pos, np.int32), dev(ref.mask_words(sees).view(np.int32)) if sees is not None else None]
        d = vbs.TreeDesc(n_q_heads=nqh, n_tokens=t, scale=hd ** -0.5, ctx_limit=limit, n_ctx=n_ctx.data_ptr(), window=140,
                         q_pos=hold[0].data_ptr(), mask=hold[1].data_ptr() if sees is not None else None,
                         k_pos=k_pos.data_ptr() if k_pos is not None else None, k_pos_per_head=int(k_pos is not None),
                         weights_out=weights.data_ptr() if weights is not None else None)
        work = torch.empty(vbs.tree_workspace(kv, d), dtype=torch.uint8, device="cuda")
        vbs.attention_tree(kv, 0, d, q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel())
        torch.cuda.synchronize()
        return out

    def store(kv, k, v, pos, slot, seq, q):
        n = k.shape[0]
        hold = [dev(pos, np.int32), dev(slot, np.int32), dev(seq, np.int32), dev(k), dev(v), dev(q)]
        out = torch.zeros(q.shape, device="cuda")
        vbs.rope_store(plan, kv, 0, hold[5].data_ptr(), out.data_ptr(), q.shape[1], hold[3].data_ptr(), hold[4].data_ptr(), n,
                       hold[0].data_ptr(), hold[1].data_ptr(), seq=hold[2].data_ptr())
        torch.cuda.synchronize()
        np.testing.assert_allclose(out.cpu().numpy(), ref.rope(q, pos, axis, hd, 10000.0, False), rtol=0, atol=ROPE_TOL)
        return out

    # the prompt, sequence by sequence interleaved
    n = S * P
    seq, slot = np.arange(n) % S, np.arange(n) // S
    pos = np.stack([slot, slot % 10], 1)
    mk = lambda n, h: rng.standard_normal((n, h, hd)).astype(np.float32)
    q = store(big, mk(n, H), mk(n, H), pos, slot, seq, mk(n, nqh))
    # the last W tokens observe the rest
    n_ctx = dev([P - W] * S, np.int32)
    weights = torch.zeros((S, H, M), device="cuda")
    qw = q.reshape(P, S, nqh, hd).transpose(0, 1)[:, P - W:].contiguous()
    q_pos = np.tile(np.arange(P - W, P), (S, 1))
    out = attention(big, n_ctx, P, qw, q_pos, weights=weights)
    rows = [x[:, 0].cpu().numpy().transpose(0, 2, 1, 3) for x in (kc, vc)]
    want, wts = ref.attend(qw.cpu().numpy(), *rows, [P - W] * S, [W] * S, hd ** -0.5, window=140, q_pos=q_pos)
    np.testing.assert_allclose(out.cpu().numpy(), want, rtol=0, atol=1e-4)
    np.testing.assert_allclose(weights.cpu().numpy(), wts, rtol=1e-5, atol=1e-4)
    # choose and move
    idx = torch.zeros((L, S, H, keep), dtype=torch.int32, device="cuda")
    count = torch.zeros((S,), dtype=torch.int32, device="cuda")
    length = dev([P] * S, np.int32)
    vbs.cache_select(weights.data_ptr(), M, L, S, H, length.data_ptr(), P, keep, 2, W, idx.data_ptr(), count.data_ptr())
    at = torch.arange(M, dtype=torch.int32, device="cuda").expand(L, S, H, M).contiguous()
    k_pos = torch.full((L, S, H, M2), -1, dtype=torch.int32, device="cuda")
    g = vbs.GatherDesc(n_max=keep, idx=idx.data_ptr(), layer_stride=S * H * keep, seq_stride=H * keep, head_stride=keep,
                       count=count.data_ptr(), pos_src=at.data_ptr(), pos_dst=k_pos.data_ptr())
    vbs.cache_gather(big, small, g)
    torch.cuda.synchronize()
    w = weights.cpu().numpy()
    for s in range(S):
        for h in range(H):
            kept = ref.select(w[s, h], P, keep, 2, W)
            assert (idx[0, s, h].cpu().numpy() == kept).all()
            assert (k_pos[0, s, h, :keep].cpu().numpy() == kept).all()
            assert (k2[s, 0, h, :keep].cpu().numpy() == rows[0][s, h, kept]).all()
    # drafts behind the kept slots; count is the new n_ctx
    trees = [ref.tree_mask(rng, T) for _ in range(S)]
    sees, depth = np.stack([t[0] for t in trees]), np.stack([t[1] for t in trees])
    seq, tok = np.arange(S * T) % S, np.arange(S * T) // S
    dpos = P + depth[seq, tok]
    q = store(small, mk(S * T, H), mk(S * T, H), np.stack([dpos, dpos % 10], 1), keep + tok, seq, mk(S * T, nqh))
    k_pos[0, :, :, keep:keep + T] = dev(P + depth, np.int32)[:, None]
    qt = q.reshape(T, S, nqh, hd).transpose(0, 1).contiguous()
    out = attention(small, count, keep + T, qt, P + depth, sees, k_pos)
    rows = [x[:, 0].cpu().numpy() for x in (k2, v2)]
    want, _ = ref.attend(qt.cpu().numpy(), *rows, [keep] * S, [T] * S, hd ** -0.5, sees=sees, window=140, q_pos=P + depth,
                         k_pos=k_pos[0].cpu().numpy())
    np.testing.assert_allclose(out.cpu().numpy(), want, rtol=0, atol=1e-4)
    # the branch to the last draft is accepted, in place
    path = [np.nonzero(sees[s, T - 1])[0] for s in range(S)]
    n_acc = [len(p) for p in path]
    lists = np.zeros((S, T), dtype=np.int32)
    for s in range(S):
        lists[s, : n_acc[s]] = path[s]
    hold = [dev(lists), dev(n_acc, np.int32)]
    g = vbs.GatherDesc(n_max=T, idx=hold[0].data_ptr(), seq_stride=T, count=hold[1].data_ptr(), src_base=count.data_ptr(),
                       dst_base=count.data_ptr(), pos_src=k_pos.data_ptr(), pos_dst=k_pos.data_ptr())
    vbs.cache_gather(small, small, g)
    torch.cuda.synchronize()
    for s in range(S):
        assert (k2[s, 0, :, keep:keep + n_acc[s]].cpu().numpy() == rows[0][s][:, keep + path[s]]).all()
        assert (v2[s, 0, :, keep:keep + n_acc[s]].cpu().numpy() == rows[1][s][:, keep + path[s]]).all()
    # one more token of each sequence
    n_ctx = count + hold[1]
    last = np.asarray([P + n_acc[s] for s in range(S)])
    q = store(small, mk(S, H), mk(S, H), np.stack([last, last % 10], 1), keep + np.asarray(n_acc), np.arange(S), mk(S, nqh))
    for s in range(S):
        k_pos[0, s, :, keep + n_acc[s]] = int(last[s])
    out = attention(small, n_ctx, M2, q.reshape(S, 1, nqh, hd), last[:, None], None, k_pos)
    rows = [x[:, 0].cpu().numpy() for x in (k2, v2)]
    want, _ = ref.attend(q.cpu().numpy().reshape(S, 1, nqh, hd), *rows, n_ctx.cpu().numpy(), [1] * S, hd ** -0.5, window=140,
                         q_pos=last[:, None], k_pos=k_pos[0].cpu().numpy())
    np.testing.assert_allclose(out.cpu().numpy(), want, rtol=0, atol=1e-4)


def test_offsets_past_32_bits(vbs, gpu):
    """Three sequences 2^31 + 8 elements apart, the last behind 2^32: store,
    attention (both kernels, with weights) and moves as in caches of their own."""
    import torch
    S, ctx, H, hd, n, stride = 3, 320, 2, 64, 300, (1 << 31) + 8
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB")
    big = [torch.empty(2 * stride + ctx * H * hd, dtype=torch.float16, device="cuda") for _ in range(2)]
    view = [[b[s * stride:s * stride + ctx * H * hd].view(ctx, H, hd) for s in range(S)] for b in big]
    for side in view:
        for x in side:
            x.fill_(0.5)
    kv = vbs.KvDesc(k=big[0].data_ptr(), v=big[1].data_ptr(), n_layers=1, max_ctx=ctx, n_kv_heads=H, head_dim=hd, n_seqs=S,
                    head_major=0, seq_stride=stride)
    rng = np.random.default_rng(1)
    x = dev(rng.standard_normal((2, S * n, H, hd)), np.float32)
    zero, slot, seq = dev(np.zeros(S * n), np.int32), dev(np.tile(np.arange(n), S), np.int32), dev(np.repeat(np.arange(S), n), np.int32)
    vbs.rope_store(vbs.rope_plan(hd), kv, 0, 0, 0, 0, x[0].data_ptr(), x[1].data_ptr(), S * n, zero.data_ptr(), slot.data_ptr(),
                   seq=seq.data_ptr())
    half = x.to(torch.float16).view(2, S, n, H, hd)
    for side in range(2):
        for s in range(S):
            assert torch.equal(view[side][s][:n], half[side, s]) and (view[side][s][n:] == 0.5).all()

    small = [torch.stack(side).contiguous() for side in view]          # the same, without gaps
    near = vbs.KvDesc(k=small[0].data_ptr(), v=small[1].data_ptr(), n_layers=1, max_ctx=ctx, n_kv_heads=H, head_dim=hd, n_seqs=S,
                      head_major=0, seq_stride=ctx * H * hd)
    for T in (1, 40):
        q = dev(rng.standard_normal((S, T, 8, hd)), np.float32)
        n_ctx = dev([n - T, 17, n - T], np.int32)
        got = []
        for c in (kv, near):
            out, w = torch.zeros_like(q), torch.zeros((S, H, ctx), device="cuda")
            t = vbs.TreeDesc(n_q_heads=8, n_tokens=T, scale=0.125, ctx_limit=ctx, n_ctx=n_ctx.data_ptr(), weights_out=w.data_ptr())
            work = torch.empty(vbs.tree_workspace(c, t), dtype=torch.uint8, device="cuda")
            vbs.attention_tree(c, 0, t, q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel())
            torch.cuda.synchronize()
            got.append((out, w))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])

    idx, count = dev(np.arange(0, n, 2), np.int32), dev([n // 2] * S, np.int32)
    g = vbs.GatherDesc(n_max=n // 2, idx=idx.data_ptr(), count=count.data_ptr())
    apart = [torch.zeros_like(s) for s in small]
    to = vbs.KvDesc(k=apart[0].data_ptr(), v=apart[1].data_ptr(), n_layers=1, max_ctx=ctx, n_kv_heads=H, head_dim=hd, n_seqs=S,
                    head_major=0, seq_stride=ctx * H * hd)
    vbs.cache_gather(kv, to, g)
    vbs.cache_gather(kv, kv, g)
    torch.cuda.synchronize()
    for side in range(2):
        for s in range(S):
            want = small[side][s][0:n:2]
            assert torch.equal(apart[side][s][:n // 2], want) and torch.equal(view[side][s][:n // 2], want)
            assert torch.equal(view[side][s][n // 2:], small[side][s][n // 2:])
