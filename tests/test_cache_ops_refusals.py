"""What the operators on a cache whose slots are not positions refuse, and
the rotary plan. No GPU: arguments are checked before any device work, and
the pointers here are never followed."""
import ctypes as C
import math

import numpy as np
import pytest

FAKE, FAR = 4096, 1 << 36


def kv(vbs, **kw):
    d = dict(k=FAKE, v=FAKE, n_layers=2, max_ctx=64, n_kv_heads=2, head_dim=64, n_seqs=2, head_major=0, seq_stride=2 * 64 * 128)
    d.update(kw)
    return vbs.KvDesc(**d)


@pytest.fixture(autouse=True)
def clean(vbs):
    vbs.clear_error()
    yield
    vbs.clear_error()


def refused(vbs, call):
    vbs.clear_error()
    with pytest.raises(vbs.VbsError, match="invalid arguments|sections of|frequency factor"):
        call()


BAD_KV = [dict(k=None), dict(v=None), dict(n_layers=0), dict(max_ctx=0), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=60),
          dict(head_dim=264), dict(n_seqs=0), dict(k=FAKE + 8), dict(seq_stride=12), dict(seq_stride=0),
          dict(seq_stride=2 * 64 * 128 - 8), dict(seq_stride=1 << 61), dict(max_ctx=0x7FFFFFFF, n_layers=1 << 31, n_seqs=1)]


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(rot_dim=12), dict(rot_dim=72),
                                dict(theta=0.0), dict(theta=-1.0), dict(theta=math.nan), dict(theta=math.inf),
                                dict(sections=[10, 10]), dict(sections=[8] * 5), dict(sections=[]),
                                dict(freq_factors=[0.0] * 32), dict(freq_factors=[math.nan] * 32)])
def test_rope_plan_refuses(vbs, kw):
    args = dict(head_dim=64)
    args.update(kw)
    refused(vbs, lambda: vbs.rope_plan(**args))


def test_rope_plan_wants_a_factor_per_pair(vbs):
    with pytest.raises(ValueError):
        vbs.rope_plan(64, freq_factors=[1.0] * 31)


def test_rope_plan_turns(vbs):
    """turn is the angle per position over 2 pi, in 2^-64: to 2^-50 of
    itself (a few roundings of doubles), cut to a whole number."""
    fac = [1.0 + 0.25 * p for p in range(48)]
    r = vbs.rope_plan(128, rot_dim=96, theta=500000.0, freq_factors=fac, sections=[16, 16, 16])
    for p in range(48):
        want = 500000.0 ** (-2.0 * p / 96) / float(np.float32(fac[p])) / (2 * math.pi) * 2.0 ** 64
        assert abs(r.turn[p] - want) <= want * 2.0 ** -50 + 1
        assert r.axis[p] == p // 16
    r = vbs.rope_plan(128, sections=[24, 20, 20], interleaved=True)
    assert [list(r.axis[:64]).count(a) for a in range(3)] == [24, 20, 20] and list(r.axis[:6]) == [0, 1, 2, 0, 1, 2]


def test_rope_store_refuses(vbs):
    plan = vbs.rope_plan(64)
    good = dict(rope=plan, kv=kv(vbs), layer=0, q=FAKE, q_out=FAKE, n_q_heads=4, k=FAKE, v=FAKE, n_tokens=1, pos=FAKE, slot=FAKE)
    for bad in ([dict(layer=2), dict(q=0), dict(q_out=0), dict(k=0), dict(v=0), dict(pos=None), dict(slot=0), dict(kv=None),
                 dict(q=FAKE + 4), dict(k=FAKE + 4), dict(q_stride=4), dict(q_stride=258), dict(kv_stride=4),
                 dict(q_stride=512), dict(rope=vbs.rope_plan(128)), dict(rope=vbs.RopeDesc()), dict(n_q_heads=0, k=0, v=0)] +
                [dict(kv=kv(vbs, **b)) for b in BAD_KV]):
        refused(vbs, lambda: vbs.rope_store(**{**good, **bad}))
    broken = vbs.rope_plan(64)
    broken.axis[5] = 1
    refused(vbs, lambda: vbs.rope_store(**{**good, "rope": broken}))


def tree(vbs, **kw):
    d = dict(n_q_heads=4, n_tokens=3, scale=0.125, ctx_limit=64, n_ctx=FAKE)
    d.update(kw)
    return vbs.TreeDesc(**d)


BAD_TREE = [dict(n_q_heads=0), dict(n_q_heads=3), dict(n_q_heads=1024), dict(n_tokens=0), dict(n_tokens=4097), dict(ctx_limit=0),
            dict(ctx_limit=65), dict(n_ctx=None), dict(scale=math.nan), dict(softcap=-1.0), dict(softcap=math.nan),
            dict(window=1 << 31), dict(weights_in=FAKE), dict(scale=math.inf), dict(softcap=math.inf), dict(softcap=1e-30)]


def test_attention_tree_refuses(vbs):
    for bad in BAD_TREE:
        refused(vbs, lambda: vbs.tree_workspace(kv(vbs), tree(vbs, **bad)))
        refused(vbs, lambda: vbs.attention_tree(kv(vbs), 0, tree(vbs, **bad), FAKE, FAR, FAKE, 1 << 30))
    for bad in BAD_KV:
        refused(vbs, lambda: vbs.tree_workspace(kv(vbs, **bad), tree(vbs)))
        refused(vbs, lambda: vbs.attention_tree(kv(vbs, **bad), 0, tree(vbs), FAKE, FAR, FAKE, 1 << 30))
    for args in ((2, FAKE, FAR, FAKE), (0, None, FAR, FAKE), (0, FAKE, None, FAKE), (0, FAKE, FAR, None),
                 (0, FAKE + 4, FAR, FAKE), (0, FAKE, FAR + 4, FAKE), (0, FAKE, FAR, FAKE + 4), (0, FAKE, FAKE, FAKE),
                 (0, FAKE, FAKE + 2 * 3 * 4 * 64 * 4 - 16, FAKE)):
        refused(vbs, lambda: vbs.attention_tree(kv(vbs), args[0], tree(vbs), *args[1:], 1 << 30))


def test_attention_tree_counts_its_limits(vbs):
    wide = kv(vbs, max_ctx=1 << 29, seq_stride=1 << 38)
    refused(vbs, lambda: vbs.tree_workspace(wide, tree(vbs, ctx_limit=(1 << 28) + 1)))
    many = kv(vbs, n_kv_heads=8192, n_seqs=1)
    refused(vbs, lambda: vbs.tree_workspace(many, tree(vbs, n_q_heads=8192 * 64, n_tokens=4096)))


def test_cache_select_refuses(vbs):
    good = dict(scores=FAKE, stride=100, n_layers=1, n_seqs=1, n_kv_heads=2, n=FAKE, n_limit=100, keep=10, first=2, recent=3,
                idx=FAKE, count=FAKE)
    for bad in (dict(scores=None), dict(n=None), dict(idx=None), dict(count=None), dict(n_layers=0), dict(n_seqs=0),
                dict(n_kv_heads=0), dict(n_limit=101), dict(keep=0), dict(first=8), dict(recent=9),
                dict(stride=1 << 22, n_limit=3145729), dict(first=0xFFFFFFFF, recent=11)):
        refused(vbs, lambda: vbs.cache_select(**{**good, **bad}))


def test_cache_gather_refuses(vbs):
    far = 1 << 40
    dst = lambda **kw: kv(vbs, **{**dict(k=far, v=2 * far), **kw})
    src = lambda **kw: kv(vbs, **{**dict(k=1 << 30, v=1 << 35), **kw})
    g = lambda **kw: vbs.GatherDesc(**{**dict(n_max=3, idx=FAKE, count=FAKE), **kw})
    for s, d, l in ([(src(), dst(n_layers=1), g()), (src(), dst(n_seqs=1), g()), (src(), dst(n_kv_heads=1), g()),
                     (src(), dst(head_dim=128), g()), (src(), dst(), g(n_max=0)), (src(), dst(), g(idx=None)),
                     (src(), dst(), g(count=None)), (src(), dst(), g(weights_src=FAKE)), (src(), dst(), g(pos_dst=FAKE)),
                     (src(), src(max_ctx=65), g()), (src(), src(v=far), g()), (src(), src(head_major=1), g()),
                     (src(), src(), g(weights_src=FAKE, weights_dst=2 * FAKE)),
                     (src(), dst(k=(1 << 30) + 256), g()), (src(), dst(v=(1 << 30) + 256), g()),
                     (src(), dst(), g(weights_src=FAKE, weights_dst=FAKE + 256))] +
                    [(src(**b), dst(), g()) for b in BAD_KV] + [(src(), dst(**b), g()) for b in BAD_KV]):
        refused(vbs, lambda: vbs.cache_gather(s, d, l))


def test_structures_match_the_header(vbs):
    assert C.sizeof(vbs.KvDesc) == 8 * 2 + 4 * 6 + 8
    assert C.sizeof(vbs.RopeDesc) == 4 * 4 + 8 * 128 + 128
    assert C.sizeof(vbs.TreeDesc) == 4 * 6 + 8 * 6 + 8 + 8 * 2
    assert C.sizeof(vbs.GatherDesc) == 8 + 8 + 8 * 3 + 8 * 7


def test_without_a_gpu_the_calls_say_so(vbs):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(vbs.VbsError, match="no usable device"):
        vbs.attention_tree(kv(vbs), 0, tree(vbs), FAKE, FAR, FAKE, 1 << 30)
