"""Buffers that one call would read and write at once are refused; neighbours
are not. No GPU: the pointers here are never followed."""
import pytest

KV, IN = 1 << 40, 1 << 32
NQ, NK, HD, N = 4, 2, 64, 5
QROW, KROW = NQ * HD * 4, NK * HD * 4     # bytes


@pytest.fixture(autouse=True)
def clean(vbs):
    vbs.clear_error()
    yield
    vbs.clear_error()


def outcome(vbs, call):
    """'' when the call ran, else the library's message ('no usable device' on a machine without one)."""
    vbs.clear_error()
    try:
        call()
    except vbs.VbsError as e:
        return str(e)
    return ""


def rope(vbs, q, q_out, k, v, q_stride=0, kv_stride=0, n=N, heads=NQ):
    kv = vbs.KvDesc(k=KV, v=KV + (1 << 30), n_layers=1, max_ctx=64, n_kv_heads=NK, head_dim=HD, n_seqs=1, head_major=0)
    return outcome(vbs, lambda: vbs.rope_store(vbs.rope_plan(HD), kv, 0, q, q_out, heads, k, v, n, 4096, 4096, q_stride=q_stride,
                                               kv_stride=kv_stride))


FUSED = (QROW + 2 * KROW) // 4            # floats of a fused q | k | v row
fused = dict(q=IN, k=IN + QROW, v=IN + QROW + KROW, q_stride=FUSED, kv_stride=FUSED)
apart = dict(q=IN, k=IN + (1 << 20), v=IN + (2 << 20))


@pytest.mark.parametrize("kw", [
    dict(apart, q_out=IN + 16), dict(apart, q_out=IN - 16), dict(apart, q_out=IN + QROW), dict(apart, q_out=IN - QROW),
    dict(apart, q_out=IN + N * QROW - 16), dict(apart, q_out=IN - N * QROW + 16),
    dict(apart, q_out=IN + (1 << 20)), dict(apart, q_out=IN + (1 << 20) - N * QROW + 16), dict(apart, q_out=IN + (1 << 20) + N * KROW - 16),
    dict(apart, q_out=IN + (2 << 20)), dict(apart, q_out=IN + (2 << 20) + N * KROW - 16),
    dict(fused, q_out=IN + QROW), dict(fused, q_out=IN + QROW + KROW), dict(fused, q_out=IN + 3 * FUSED * 4 + 16),
    dict(fused, q_out=IN - N * QROW + 16), dict(fused, q_out=IN + (N - 1) * FUSED * 4 + QROW),
    dict(fused, q_out=IN + QROW, q_stride=1 << 40, kv_stride=1 << 62)])
def test_rope_store_refuses_a_result_over_its_inputs(vbs, kw):
    assert "invalid arguments" in rope(vbs, **kw)


@pytest.mark.parametrize("kw", [
    dict(apart, q_out=IN), dict(apart, q_out=IN + N * QROW), dict(apart, q_out=IN - N * QROW),
    dict(apart, q_out=IN + (1 << 20) + N * KROW), dict(apart, q_out=IN + (1 << 20) - N * QROW), dict(apart, q_out=IN, n=0),
    dict(apart, q_out=IN + 16, n=0), dict(fused, q_out=IN - N * QROW), dict(fused, q_out=IN + N * FUSED * 4),
    dict(fused, q_out=IN + FUSED * 4 - 2 * KROW, n=1, k=IN + (1 << 20), v=IN + (2 << 20)),
    # rows so far apart that the whole result fits between two of them
    dict(apart, q_stride=1 << 16, k=IN + (8 << 20), v=IN + (9 << 20), q_out=IN + QROW),
    dict(apart, q_stride=1 << 16, k=IN + (8 << 20), v=IN + (9 << 20), q_out=IN + (1 << 18) * 2 - N * QROW),
    dict(q=0, q_out=0, heads=0, k=IN, v=IN)])
def test_rope_store_takes_what_does_not_overlap(vbs, kw):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: the call would run")
    got = rope(vbs, **kw)
    assert "no usable device" in got


W = 2 * NK * 64 * 4                       # bytes of the weights: sequences, heads, max_ctx


@pytest.mark.parametrize("shift,fine", [(0, True), (W, True), (-W, True), (16, False), (-16, False), (W - 16, False), (16 - W, False)])
def test_attention_weights_in_over_weights_out(vbs, shift, fine):
    """The same buffer, or none of it: each position's sum is read and written
    by a thread of its own."""
    import torch
    if fine and torch.cuda.is_available():
        pytest.skip("a GPU is present: the call would run")
    kv = vbs.KvDesc(k=KV, v=KV + (1 << 30), n_layers=1, max_ctx=64, n_kv_heads=NK, head_dim=HD, n_seqs=2, head_major=0, seq_stride=64 * NK * HD)
    tree = vbs.TreeDesc(n_q_heads=NQ, n_tokens=3, scale=0.125, ctx_limit=64, n_ctx=4096, weights_in=IN + shift, weights_out=IN)
    for call in (lambda: vbs.tree_workspace(kv, tree),
                 lambda: vbs.attention_tree(kv, 0, tree, IN + (1 << 20), IN + (2 << 20), IN + (3 << 20), 1 << 20)):
        assert ("no usable device" if fine else "invalid arguments") in outcome(vbs, call)
